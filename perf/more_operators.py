"""Measured cases of linear attention with a decay for each head (whole sequences, training, single
tokens of cached streams) and of the group norm with an activation and a gate that follows it in a
retention layer and in convolutional heads.

Per sequence and head, with lambda = exp(log_decay) (state S [key dim, value dim], zeros or the given
one before the first token):

    linear attention   S_t = lambda S_{t-1} + k_t v_t^T          o_t = scale q_t^T S_t

Group norm, over the channels of a group and (images) all pixels, or (rows) one row by itself:

    n = (x - mean) / sqrt(var + eps) * weight + bias             y = act(n) * silu(gate)
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CHUNK = 64


def listed():
    return [
        # one token of one stream: the latency of the smallest call
        dict(name="step_one", op="step", type="bf16", batch=1, slots=1, heads=8, key=64, value=64),
        # a serving batch that advances 256 of 320 cached streams by a token
        dict(name="step_batch", op="step", type="bf16", batch=256, slots=320, heads=16, key=128, value=128),
        # ragged prompts, packed, that continue cached states; values twice as wide as keys
        dict(name="prompts", op="linear", type="bf16", batch=24, length=16384, heads=8, key=64, value=128, ragged=True,
             train=False, reverse=False),
        # dense-prediction tokens (64 x 256) of two images: few chains, each of them long
        dict(name="rows_64x256", op="linear", type="bf16", batch=2, length=16384, heads=4, key=64, value=64, ragged=False,
             train=False, reverse=False),
        # long sequences with many wide heads
        dict(name="long_prompts", op="linear", type="bf16", batch=4, length=8192, heads=16, key=128, value=128,
             ragged=False, train=False, reverse=False),
        # a training step on second-stage images (28 x 28 tokens, 128 channels expanded twice), batch 64
        dict(name="train_28x28", op="linear", type="bf16", batch=64, length=784, heads=4, key=64, value=64, ragged=False,
             train=True, reverse=False),
        # odd sizes in fp32, read from the last token to the first, as a bidirectional mixer does
        dict(name="train_odd", op="linear", type="fp32", batch=3, length=785, heads=5, key=48, value=72, ragged=False,
             train=True, reverse=True),
        # the tokens of a serving batch behind the attention: every row by itself, a group a head, gated
        dict(name="norm_step", op="rows", type="bf16", rows=256, channels=2048, groups=16, activation="", gate=True,
             train=False),
        # the rows of 64 second-stage images behind the attention, training
        dict(name="norm_rows_train", op="rows", type="bf16", rows=50176, channels=256, groups=4, activation="", gate=True,
             train=True),
        # one last-stage image in fp32
        dict(name="norm_7x7", op="image", type="fp32", batch=1, height=7, width=7, channels=768, groups=32,
             activation="silu", gate=False, train=False),
        # first-stage maps of two wide images (128 x 512), as a dense-prediction head normalises them
        dict(name="norm_128x512", op="image", type="bf16", batch=2, height=128, width=512, channels=128, groups=32,
             activation="gelu", gate=False, train=False),
        # a training step on first-stage images, batch 64
        dict(name="norm_train_56x56", op="image", type="bf16", batch=64, height=56, width=56, channels=128, groups=32,
             activation="silu", gate=False, train=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "step", "rows", "image", "image"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    if op == "step":
        key, value = rng.choice([(32, 32), (64, 64), (64, 128), (128, 128), (40, 72)])
        batch = _spread(rng, 1, 256)
        return dict(op=op, type=kind, batch=batch, slots=batch + rng.randrange(0, 64), heads=rng.randrange(1, 17), key=key,
                    value=value)
    if op == "linear":
        key, value = rng.choice([(16, 16), (32, 32), (64, 64), (64, 64), (64, 128), (128, 128), (128, 128), (48, 72),
                                 (100, 60)])
        ragged = rng.random() < 0.4
        while True:
            batch, length, heads = _spread(rng, 1, 64), _spread(rng, 16, 16384), _spread(rng, 1, 16)
            # a pass of the plain form stays under the largest listed one's: tokens by head width, and chunks squared
            rows = length * (1 if ragged else batch)
            if rows * heads * (key + value) <= (24_000_000 if train or kind == "fp32" else 64_000_000) and rows <= 60_000:
                break
        return dict(op=op, type=kind, batch=batch, length=length, heads=heads, key=key, value=value, ragged=ragged,
                    train=train, reverse=rng.random() < 0.3)
    activation, gate = rng.choice(["", "silu", "gelu"]), rng.random() < 0.4
    per, groups = rng.choice([(2, 32), (3, 32), (4, 32), (8, 32), (24, 32), (64, 4), (128, 8), (60, 5), (96, 1), (1, 96), (13, 7)])
    if op == "rows":
        per, groups = rng.choice([(24, 32), (64, 4), (64, 16), (128, 8), (128, 16), (60, 5), (96, 1), (256, 4), (50, 7)])
    case = dict(type=kind, channels=per * groups, groups=groups, activation=activation, gate=gate, train=train)
    if op == "rows":
        return dict(op=op, rows=_spread(rng, 1, 12_000_000 // (per * groups)), **case)
    while True:
        batch, height, width = _spread(rng, 1, 128), _spread(rng, 1, 128), _spread(rng, 1, 512)
        # a group of a handful of values says little: its gradient is what is left of a difference
        if batch * height * width * per * groups <= 25_000_000 and height * width * per >= 32:
            break
    return dict(op=op, batch=batch, height=height, width=width, **case)


def _cuts(case, seed):
    """Offsets of ``batch`` packed sequences over ``length`` tokens, some empty or one token long."""
    rng, total, count = random.Random(seed), case["length"], case["batch"]
    cuts = sorted(rng.randrange(0, total + 1) for _ in range(count - 1))
    if count >= 4:
        cuts[1] = cuts[0]                      # a sequence without tokens
        cuts[2] = max(cuts[2], cuts[1])
    if count >= 5:
        cuts[3] = min(total, cuts[2] + 1)      # a sequence of one token
        cuts[4:] = [max(c, cuts[3]) for c in cuts[4:]]
    return [0] + cuts + [total]


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), _TYPES[case["type"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    train = bool(case.get("train"))

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).add_(shift)

    def given(t):
        return t.requires_grad_() if train else t

    s = dict(case=case)
    if case["op"] in ("rows", "image"):
        c = case["channels"]
        if case["op"] == "rows":
            x = normal(case["rows"], c, scale=2.0, shift=0.5).to(dtype)
            gate = normal(case["rows"], 2 * c).to(dtype)[:, c:] if case["gate"] else None   # half of a projection
        else:
            shape = case["batch"], case["height"], case["width"], c
            x = normal(*shape, scale=2.0, shift=0.5).to(dtype).permute(0, 3, 1, 2)
            gate = normal(*shape).to(dtype).permute(0, 3, 1, 2) if case["gate"] else None
        s["x"], s["gate"] = given(x), None if gate is None else given(gate)
        s["weight"], s["bias"] = given(normal(c, scale=0.2, shift=1.0)), given(normal(c, scale=0.2))
        if train:
            s["dy"] = torch.empty_like(x).copy_(normal(*x.shape))
        return s
    h, dk, dv = case["heads"], case["key"], case["value"]
    # decays of 1 - 2^-2 (a window of 4 tokens) to 1 - 2^-9, spread over the heads
    s["log_decay"] = torch.log1p(-torch.exp2(-2.0 - 7.0 * torch.arange(h, device=dev, dtype=torch.float32) / max(1, h - 1)))
    s["scale"] = 1.0 / math.sqrt(dk)
    if case["op"] == "step":
        lead = (case["batch"],)
        s["slots"] = torch.randperm(case["slots"], generator=gen, device=dev)[:case["batch"]].to(torch.int32)
        s["state"] = normal(case["slots"], h, dk, dv)
        s["state_out"] = s["state"].clone()
    elif case["ragged"]:
        lead = (case["length"],)
        s["cuts"] = _cuts(case, seed)
        s["offsets"] = torch.tensor(s["cuts"], dtype=torch.int32, device=dev)
        s["initial"] = given(normal(case["batch"], h, dk, dv))
    else:
        lead = (case["batch"], case["length"])
        s["offsets"], s["initial"] = None, None
    # queries, keys and values leave one projection
    rows = normal(*lead, h * (2 * dk + dv)).to(dtype)
    s["q"] = given(rows[..., :h * dk].view(*lead, h, dk))
    s["k"] = given(rows[..., h * dk:2 * h * dk].view(*lead, h, dk))
    s["v"] = given(rows[..., 2 * h * dk:].view(*lead, h, dv))
    if train:
        s["do"] = normal(*lead, h, dv).to(dtype)
    return s


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        if case["op"] == "step":
            return _plain_step(state)
        return _plain_norm(state, case) if case["op"] in ("rows", "image") else _plain_linear(state, case)


# ---- the framework's operators ------------------------------------------------------------------
def _run_own(s, case):
    if case["op"] in ("rows", "image"):
        from visionhope_b200.utils.group_norm import group_norm, group_norm_rows

        norm = group_norm_rows if case["op"] == "rows" else group_norm
        y = norm(s["x"], case["groups"], s["weight"], s["bias"], 1e-5, activation=case["activation"] or None, gate=s["gate"])
        out, loss, names = {"y": y}, y, ("x", "gate", "weight", "bias")
    else:
        from visionhope_b200.ssm_core import linear_attention, linear_attention_step

        if case["op"] == "step":
            o = linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"], slots=s["slots"],
                                      state_out=s["state_out"])
            return {"o": o, "state": s["state_out"]}
        got = linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], initial_state=s["initial"],
                               return_final_state=case["ragged"], seq_offsets=s["offsets"], reverse=case["reverse"])
        out = {"o": got[0], "state": got[1]} if case["ragged"] else {"o": got}
        loss, names = out["o"], ("q", "k", "v", "initial")
    if case["train"]:
        names = [k for k in names if s[k] is not None]
        grads = torch.autograd.grad(loss, [s[k] for k in names], s["do"] if "do" in s else s["dy"])
        out.update(("d_" + k, g) for k, g in zip(names, grads))
    return out


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end -------------------
def _plain_norm(s, case):
    x, c, g = s["x"].float(), case["channels"], case["groups"]
    lay = (lambda t: t[:, None, :]) if case["op"] == "rows" else (lambda t: t.permute(0, 2, 3, 1).flatten(1, 2))
    unlay = (lambda t: t[:, 0]) if case["op"] == "rows" else (
        lambda t: t.unflatten(1, (case["height"], case["width"])).permute(0, 3, 1, 2))
    x = lay(x)                                                               # [samples, pixels, channels]
    n, p, _ = x.shape
    xg = x.reshape(n, p, g, c // g)
    mean = xg.mean((1, 3), keepdim=True)
    xc = xg - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
    xhat = (xc * rstd).view(n, p, c)
    pre = xhat * s["weight"] + s["bias"]
    act, slope = pre, torch.ones_like(pre)
    if case["activation"] == "silu":
        sig = 1.0 / (1.0 + torch.exp(-pre))
        act, slope = pre * sig, sig * (1.0 + pre * (1.0 - sig))
    elif case["activation"] == "gelu":
        phi = 0.5 * (1.0 + torch.erf(pre * math.sqrt(0.5)))
        act, slope = pre * phi, phi + pre * torch.exp(-0.5 * pre * pre) * (1.0 / math.sqrt(2.0 * math.pi))
    y, z = act, None
    if s["gate"] is not None:
        z = lay(s["gate"].float())
        sz = 1.0 / (1.0 + torch.exp(-z))
        y = act * z * sz
    out = {"y": unlay(y).to(s["x"].dtype)}
    if case["train"]:
        dy = lay(s["dy"].float())
        if z is not None:
            out["d_gate"] = unlay(dy * act * sz * (1.0 + z * (1.0 - sz))).to(s["x"].dtype)
            dy = dy * z * sz
        dn = dy * slope
        out["d_weight"], out["d_bias"] = (dn * xhat).sum((0, 1)), dn.sum((0, 1))
        dh, hg = (dn * s["weight"]).view(n, p, g, c // g), xhat.view(n, p, g, c // g)
        dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - hg * (dh * hg).mean((1, 3), keepdim=True))
        out["d_x"] = unlay(dx.reshape(n, p, c)).to(s["x"].dtype)
    return out


def _chunks(s, case, reverse, device):
    """Chunks of at most _CHUNK tokens: the row of each place in each chunk ([chunks, _CHUNK]), which places
    hold a token, each chunk's sequence and its first and end token within it; and the tokens of each sequence."""
    if s["offsets"] is None:
        starts = torch.arange(case["batch"] + 1, device=device) * case["length"]
        most = case["batch"] * (-(-case["length"] // _CHUNK))
    else:
        starts = s["offsets"].long()
        most = case["length"] // _CHUNK + case["batch"]
    count = starts[1:] - starts[:-1]
    cum = torch.cumsum((count + _CHUNK - 1) // _CHUNK, 0)
    at = torch.arange(most, device=device)
    seq = torch.searchsorted(cum, at, right=True).clamp(max=count.numel() - 1)
    before = cum - (count + _CHUNK - 1) // _CHUNK
    place = (at - before[seq])[:, None] * _CHUNK + torch.arange(_CHUNK, device=device)
    live = (place < count[seq][:, None]) & (at < cum[-1])[:, None]
    rows = starts[seq][:, None] + (count[seq][:, None] - 1 - place if reverse else place)
    first = place[:, 0]
    end = torch.minimum(first + _CHUNK, count[seq])
    return torch.where(live, rows, torch.zeros_like(rows)), live, seq, first, end, count


def _plain_attend(q, k, v, g, initial, where, scale):
    """o (rows as q's) and the final states of the chunked form; q, k, v fp32 [rows, heads, dim]."""
    rows, live, seq, first, end, count = where
    off = lambda t: (t[rows] * live[:, :, None, None]).transpose(1, 2)       # [chunks, heads, _CHUNK, dim]  # noqa: E731
    qc, kc, vc = off(q), off(k), off(v)
    at = torch.arange(_CHUNK, device=q.device)
    ahead = at[:, None] - at[None, :]
    mask = torch.where(ahead >= 0, torch.exp(g[:, None, None] * ahead.clamp(min=0)), torch.zeros((), device=q.device))
    o = (qc @ kc.transpose(-1, -2) * mask) @ vc
    # each chunk's own state at its end, then what reaches each chunk's start from the ones before it
    left = (end - first)[:, None] - 1 - at
    weight = torch.where(left >= 0, torch.exp(g[:, None, None] * left.clamp(min=0)), torch.zeros((), device=q.device))
    own_state = (kc * weight.transpose(0, 1)[..., None]).transpose(-1, -2) @ vc   # [chunks, heads, key, value]
    gap = first[:, None] - end[None, :]
    used = live[:, 0]
    joined = (seq[:, None] == seq[None, :]) & (gap >= 0) & used[:, None] & used[None, :]
    reach = torch.where(joined, torch.exp(g[:, None, None] * gap.clamp(min=0)), torch.zeros((), device=q.device))
    n, h, dk, dv = own_state.shape
    flat = own_state.transpose(0, 1).reshape(h, n, dk * dv)
    state = (reach @ flat).view(h, n, dk, dv).transpose(0, 1)
    if initial is not None:
        state = state + torch.exp(g * first[:, None])[..., None, None] * initial[seq]
    o = o + (qc * torch.exp(g[:, None] * (at + 1))[..., None]) @ state
    out = torch.zeros(q.shape[0], h, dv, device=q.device)
    out[rows[live]] = o.transpose(1, 2)[live] * scale
    # the state after the last token of every sequence
    gap = count[:, None] - end[None, :]
    joined = (torch.arange(count.numel(), device=q.device)[:, None] == seq[None, :]) & used[None, :]
    reach = torch.where(joined, torch.exp(g[:, None, None] * gap.clamp(min=0)), torch.zeros((), device=q.device))
    final = (reach @ flat).view(h, -1, dk, dv).transpose(0, 1)
    if initial is not None:
        final = final + torch.exp(g * count[:, None])[..., None, None] * initial
    return out, final


def _plain_linear(s, case):
    shape, dtype, g, scale = s["q"].shape, s["q"].dtype, s["log_decay"], s["scale"]
    q, k, v = (s[n].float().reshape(-1, case["heads"], s[n].shape[-1]) for n in ("q", "k", "v"))
    ahead = _chunks(s, case, case["reverse"], q.device)
    o, final = _plain_attend(q, k, v, g, s["initial"], ahead, scale)
    out = {"o": o.view(*shape[:-1], -1).to(dtype)}
    if case["ragged"]:
        out["state"] = final
    if case["train"]:
        # each gradient is such an attention itself: dq_i = sum_j<=i lambda^(i-j) (do_i v_j) k_j, and dk, dv the
        # same from the last token to the first
        do = s["do"].float().reshape(-1, case["heads"], v.shape[-1])
        back = _chunks(s, case, not case["reverse"], q.device)
        initial = None if s["initial"] is None else s["initial"].transpose(-1, -2)
        dq, _ = _plain_attend(do, v, k, g, initial, ahead, scale)
        dk, _ = _plain_attend(v, do, q, g, None, back, scale)
        dv, carried = _plain_attend(k, q, do, g, None, back, scale)
        out.update(d_q=dq.view(shape).to(dtype), d_k=dk.view(shape).to(dtype), d_v=dv.view(s["v"].shape).to(dtype))
        if initial is not None:
            # what reaches the state before the first token: the carried state, one decay further
            out["d_initial"] = scale * torch.exp(g)[:, None, None] * carried
    return out


def _plain_step(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    at = s["slots"].long()
    state = torch.exp(s["log_decay"])[:, None, None] * s["state"][at] + k[..., :, None] * v[..., None, :]
    o = s["scale"] * (q[..., :, None] * state).sum(-2)
    s["state_out"][at] = state
    return {"o": o.to(s["q"].dtype), "state": s["state_out"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rows", "image"):
        return _exact_norm(s, case)
    with torch.no_grad():
        v = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
        return _exact_step(s, v) if case["op"] == "step" else _exact_linear(s, v, case)


def _exact_norm(s, case):
    """The definition under autograd."""
    names = [k for k in ("x", "gate", "weight", "bias") if s[k] is not None]
    with torch.enable_grad():
        v = {k: s[k].detach().double().requires_grad_() for k in names}
        c, g = case["channels"], case["groups"]
        x, per = v["x"], (1, c) + (1,) * (v["x"].dim() - 2)
        xg = x.reshape(x.shape[0], g, -1)
        var, mean = torch.var_mean(xg, dim=2, unbiased=False, keepdim=True)
        y = ((xg - mean) / (var + 1e-5).sqrt()).reshape(x.shape) * v["weight"].view(per) + v["bias"].view(per)
        if case["activation"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["activation"] == "gelu":
            y = 0.5 * y * torch.erfc(-y / math.sqrt(2.0))
        if s["gate"] is not None:
            y = y * v["gate"] * torch.sigmoid(v["gate"])
        out = {"y": y.detach()}
        if case["train"]:
            out.update(("d_" + k, t) for k, t in zip(names, torch.autograd.grad(y, [v[k] for k in names], s["dy"].double())))
    return out


def _exact_step(s, v):
    state, at = v["state"].clone(), s["slots"].long()
    state[at] = torch.einsum("h,bhkv->bhkv", v["log_decay"].exp(), state[at]) + torch.einsum("bhk,bhv->bhkv", v["k"], v["v"])
    return {"o": s["scale"] * torch.einsum("bhk,bhkv->bhv", v["q"], state[at]), "state": state}


def _exact_linear(s, v, case):
    """Token by token, all sequences side by side."""
    cuts = s["cuts"] if s["offsets"] is not None else [i * case["length"] for i in range(case["batch"] + 1)]
    h, dk, dv = case["heads"], case["key"], case["value"]
    first = torch.tensor(cuts[:-1], device=v["q"].device)
    count = torch.tensor(cuts[1:], device=v["q"].device) - first
    longest = max(b - a for a, b in zip(cuts[:-1], cuts[1:]))
    q, k, val = v["q"].reshape(-1, h, dk), v["k"].reshape(-1, h, dk), v["v"].reshape(-1, h, dv)
    do = v["do"].reshape(-1, h, dv) if case["train"] else None
    decay = v["log_decay"].exp().view(1, h, 1, 1)
    state = torch.zeros(len(first), h, dk, dv, dtype=torch.float64, device=q.device) if s["initial"] is None else v["initial"].clone()
    order = sorted(range(len(first)), key=lambda i: cuts[i] - cuts[i + 1])   # longest first: the live ones lead
    perm = torch.tensor(order, device=q.device)
    lengths = [cuts[i + 1] - cuts[i] for i in order]
    state, first, count = state[perm], first[perm], count[perm]
    alive, here = [0] * longest, len(order)
    for t in range(longest):
        while here and lengths[here - 1] <= t:
            here -= 1
        alive[t] = here
    at = lambda t, n: first[:n] + (count[:n] - 1 - t if case["reverse"] else t)  # noqa: E731
    o, dq = torch.zeros_like(val), torch.zeros_like(q)
    for t in range(longest):
        n = alive[t]
        r = at(t, n)
        state[:n] = decay * state[:n] + k[r].unsqueeze(-1) * val[r].unsqueeze(-2)
        o[r] = (q[r].unsqueeze(-2) @ state[:n]).squeeze(-2)
        if do is not None:
            dq[r] = (state[:n] @ do[r].unsqueeze(-1)).squeeze(-1)
    back = torch.empty_like(perm)
    back[perm] = torch.arange(len(order), device=perm.device)
    out = {"o": s["scale"] * o.view(*s["q"].shape[:-1], dv)}
    if case["ragged"]:
        out["state"] = state[back]
    if do is None:
        return out
    dk_, dv_, ds = torch.zeros_like(k), torch.zeros_like(val), torch.zeros_like(state)
    for t in reversed(range(longest)):
        n = alive[t]
        r = at(t, n)
        ds[:n] = ds[:n] + q[r].unsqueeze(-1) * do[r].unsqueeze(-2)
        dk_[r] = (ds[:n] @ val[r].unsqueeze(-1)).squeeze(-1)
        dv_[r] = (k[r].unsqueeze(-2) @ ds[:n]).squeeze(-2)
        ds[:n] = decay * ds[:n]
    out.update((n, s["scale"] * g.view(like.shape)) for n, g, like in
               (("d_q", dq, s["q"]), ("d_k", dk_, s["k"]), ("d_v", dv_, s["v"])))
    if s["initial"] is not None:
        out["d_initial"] = s["scale"] * ds[back]
    return out


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] in ("rows", "image"):
        n = case["channels"] * (case["rows"] if case["op"] == "rows" else case["batch"] * case["height"] * case["width"])
        tensors = (2 + case["gate"]) + (2 + case["gate"] if case["train"] else 0)   # forward; dy, dx and the gate's
        return {"bytes": n * size * tensors + 4 * case["channels"] * (4 if case["train"] else 2),
                "flops": n * (30 if case["train"] else 10)}
    h, dk, dv = case["heads"], case["key"], case["value"]
    if case["op"] == "step":
        return {"bytes": case["batch"] * h * (8 * dk * dv + size * (2 * dk + 2 * dv)), "flops": 5 * case["batch"] * h * dk * dv}
    rows = case["length"] * (1 if case["ragged"] else case["batch"])
    data = rows * h * (2 * dk + 2 * dv) * size
    states = 8 * case["batch"] * h * dk * dv if case["ragged"] else 0
    if case["train"]:
        data += rows * h * (2 * dk + 2 * dv) * size                           # do, and three gradients
        states += 4 * case["batch"] * h * dk * dv if case["ragged"] else 0
    # the recurrence: an update and a product of the state a token; backward both states and three products
    return {"bytes": data + states, "flops": rows * h * dk * dv * (14 if case["train"] else 4)}
