"""Measured cases of the selective state space operators: the short causal convolution and the
selective scan, over whole sequences (prompts, images read as token rows, training) and for single
tokens (a cache of states that advances one token a call).

All sequences are channels-last, ``[batch, length, channels]``, or packed ``[tokens, channels]`` with
``offsets`` that say where each sequence starts.  The formulas, per sequence, channel d and state n:

    convolution   c_t = bias_d + sum_k w_{d,k} x_{t-K+1+k},   y_t = c_t or silu(c_t)
    scan          s_t = softplus(delta_t + delta_bias_d)
                  h_t = exp(s_t A_{d,n}) h_{t-1} + s_t u_t B_{t,n}
                  y_t = (sum_n C_{t,n} h_t + D_d u_t) silu(z_t)

The values before a sequence's first token are its initial state (zeros without one).
"""
import math
import random

import torch
import torch.nn.functional as F

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token of one stream through the convolution: the latency of the smallest call
        dict(name="conv_step_one", op="conv_step", type="bf16", batch=1, slots=1, channels=512, taps=4),
        # a serving batch that advances 256 of 320 cached streams by a token
        dict(name="conv_step_batch", op="conv_step", type="bf16", batch=256, slots=320, channels=2048, taps=4),
        # ragged prompts, packed, that continue cached states
        dict(name="conv_prompts", op="conv", type="bf16", batch=24, length=16384, channels=1024, taps=4, ragged=True,
             train=False, reverse=False),
        # a training step on first-stage images (56 x 56 tokens, 64 channels expanded twice), batch 64
        dict(name="conv_train_56x56", op="conv", type="bf16", batch=64, length=3136, channels=128, taps=4, ragged=False,
             train=True, reverse=False),
        # odd sizes in fp32, read from the last token to the first, as a bidirectional mixer does
        dict(name="conv_train_odd", op="conv", type="fp32", batch=3, length=785, channels=250, taps=3, ragged=False,
             train=True, reverse=True),
        # one token of one stream through the scan
        dict(name="scan_step_one", op="scan_step", type="bf16", batch=1, slots=1, channels=512, states=16),
        # a serving batch that advances 256 of 320 cached streams by a token
        dict(name="scan_step_batch", op="scan_step", type="bf16", batch=256, slots=320, channels=2048, states=16),
        # third-stage images (14 x 14 tokens, 256 channels expanded twice) in fp32, inference
        dict(name="scan_14x14", op="scan", type="fp32", batch=8, length=196, channels=512, states=16, groups=1,
             ragged=False, train=False, reverse=False),
        # dense-prediction tokens (64 x 256) of two images: few chains, each of them long
        dict(name="scan_64x256", op="scan", type="bf16", batch=2, length=16384, channels=384, states=16, groups=1,
             ragged=False, train=False, reverse=False),
        # ragged prompts, packed, that continue cached states
        dict(name="scan_prompts", op="scan", type="bf16", batch=17, length=8192, channels=1024, states=16, groups=1,
             ragged=True, train=False, reverse=False),
        # a training step on second-stage images (28 x 28 tokens, 128 channels expanded twice), batch 64
        dict(name="scan_train_28x28", op="scan", type="bf16", batch=64, length=784, channels=256, states=16, groups=1,
             ragged=False, train=True, reverse=False),
        # a training step on long rows with odd sizes, two groups of B and C, in reverse
        dict(name="scan_train_long", op="scan", type="bf16", batch=2, length=4095, channels=190, states=16, groups=2,
             ragged=False, train=True, reverse=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op.endswith("step"):
        batch = _spread(rng, 1, 256)
        case = dict(op=op, type=kind, batch=batch, slots=batch + rng.randrange(0, 64), channels=_spread(rng, 64, 2048))
        case.update(dict(taps=rng.choice([2, 3, 4])) if op == "conv_step" else dict(states=rng.choice([8, 16, 16])))
        return case
    train, ragged = rng.random() < 0.5, rng.random() < 0.4
    groups = rng.choice([1, 1, 2]) if op == "scan" else 1
    while True:
        batch, length = _spread(rng, 1, 64), _spread(rng, 16, 16384)
        channels = groups * _spread(rng, 16, 1024 // groups)
        elements = channels * length * (1 if ragged else batch)
        if elements <= (25_000_000 if op == "conv" else 8_000_000):
            break
    case = dict(op=op, type=kind, batch=batch, length=length, channels=channels, ragged=ragged, train=train,
                reverse=rng.random() < 0.3)
    case.update(dict(taps=rng.choice([2, 3, 4])) if op == "conv"
                else dict(states=rng.choice([8, 16, 16, 16]), groups=groups))
    return case


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
    d = case["channels"]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).add_(shift)

    state = dict(case=case)
    if case["op"].endswith("step"):
        batch, slots = case["batch"], case["slots"]
        lead = (batch,)
        order = torch.randperm(slots, generator=gen, device=dev)[:batch]
        state["slots"] = order.to(torch.int32)
    elif case["ragged"]:
        lead = (case["length"],)
        cuts = _cuts(case, seed)
        state["cuts"] = cuts
        state["offsets"] = torch.tensor(cuts, dtype=torch.int32, device=dev)
    else:
        lead = (case["batch"], case["length"])
        state["offsets"] = None
    train = bool(case.get("train"))

    def given(t):
        return t.requires_grad_() if train else t

    # the two halves of one input projection: the token rows are 2 d apart
    halves = normal(*lead, 2 * d).to(dtype)
    x, z = halves[..., :d], halves[..., d:]
    if case["op"].startswith("conv"):
        k = case["taps"]
        state["x"] = given(x)
        state["weight"] = given(normal(d, k, scale=1.0 / math.sqrt(k)))
        state["bias"] = given(normal(d, scale=0.1))
        if case["op"] == "conv_step":
            state["state"] = normal(case["slots"], k - 1, d).to(dtype)
            state["state_out"] = state["state"].clone()
        elif case["ragged"]:
            state["initial"] = given(normal(case["batch"], k - 1, d).to(dtype))
        else:
            state["initial"] = None
    else:
        n, groups = case["states"], case.get("groups", 1)
        rank = max(1, d // 32)
        # delta, B and C leave one projection; delta then goes through a second one
        rows = normal(*lead, rank + 2 * groups * n).to(dtype)
        bc = rows[..., rank:].view(*lead, 2, groups, n) if groups > 1 else rows[..., rank:].view(*lead, 2, n)
        b, c = (bc[..., 0, :, :], bc[..., 1, :, :]) if groups > 1 else (bc[..., 0, :], bc[..., 1, :])
        state["u"] = given(F.silu(normal(*lead, d)).to(dtype))
        state["z"] = given(z)
        state["delta"] = given(normal(*lead, d, scale=0.5).to(dtype))
        state["B"], state["C"] = given(b), given(c)
        state["A"] = given(-torch.arange(1, n + 1, device=dev, dtype=torch.float32).repeat(d, 1)
                           * torch.exp(normal(d, n, scale=0.1)))
        state["D"] = given(normal(d, scale=0.1, shift=1.0))
        # softplus(delta_bias) between 0.001 and 0.1, spread over its logarithm
        step = torch.exp(torch.rand(d, generator=gen, device=dev) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        state["delta_bias"] = given(step + torch.log(-torch.expm1(-step)))
        if case["op"] == "scan_step":
            state["state"] = normal(case["slots"], d, n)
            state["state_out"] = state["state"].clone()
        elif case["ragged"]:
            state["initial"] = given(normal(case["batch"], d, n))
        else:
            state["initial"] = None
    if train:
        state["dy"] = normal(*lead, d).to(dtype)
    return state


_CONV_INPUTS = ("x", "weight", "bias", "initial")
_SCAN_INPUTS = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial")


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "conv_step":
        return _plain_conv_step(state)
    if case["op"] == "scan_step":
        return _plain_scan_step(state)
    with torch.no_grad():
        return _plain_conv(state, case) if case["op"] == "conv" else _plain_scan(state, case)


# ---- the framework's operators ------------------------------------------------------------------
def _run_own(s, case):
    from visionhope_b200.ssm_core import short_conv, short_conv_step, ssm_scan, ssm_scan_step

    if case["op"] == "conv_step":
        y = short_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu", slots=s["slots"],
                            state_out=s["state_out"])
        return {"y": y, "state": s["state_out"]}
    if case["op"] == "scan_step":
        y = ssm_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                          delta_bias=s["delta_bias"], delta_softplus=True, slots=s["slots"], state_out=s["state_out"])
        return {"y": y, "state": s["state_out"]}
    want = case["ragged"]
    if case["op"] == "conv":
        names = _CONV_INPUTS
        got = short_conv(s["x"], s["weight"], s["bias"], activation="silu", initial_state=s["initial"],
                         return_final_state=want, seq_offsets=s["offsets"], reverse=case["reverse"])
    else:
        names = _SCAN_INPUTS
        got = ssm_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                       delta_softplus=True, initial_state=s["initial"], return_final_state=want,
                       seq_offsets=s["offsets"], reverse=case["reverse"])
    y, final = got if want else (got, None)
    out = {"y": y} if final is None else {"y": y, "state": final}
    if case["train"]:
        names = [k for k in names if s[k] is not None]
        out.update(("d_" + k, g) for k, g in zip(names, torch.autograd.grad(y, [s[k] for k in names], s["dy"])))
    return out


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end -------------------
def _wide(s, *names):
    return [None if s.get(k) is None else s[k].float() for k in names]


def _silu_grad(c):
    sig = torch.sigmoid(c)
    return sig * (1.0 + c * (1.0 - sig))


def _order(s, case, device):
    """Rows of the token axis in scan order, and which sequence each belongs to: both [tokens]."""
    if s["offsets"] is None:
        batch, length = case["batch"], case["length"]
        starts = torch.arange(batch + 1, device=device) * length
    else:
        starts = s["offsets"].long()
    total = case["length"] if s["offsets"] is not None else case["batch"] * case["length"]
    at = torch.arange(total, device=device)
    seq = torch.searchsorted(starts[1:], at, right=True)
    rows = starts[seq] + starts[seq + 1] - 1 - at if case["reverse"] else at
    return rows, seq, starts


def _plain_conv(s, case):
    x, w, bias, initial, dy = _wide(s, "x", "weight", "bias", "initial", "dy")
    dtype, shape, d, k = s["x"].dtype, x.shape, case["channels"], case["taps"]
    rows, seq, starts = _order(s, case, x.device)
    x, count, total = x.reshape(-1, d)[rows], starts.numel() - 1, rows.numel()
    if initial is None:
        initial = torch.zeros(count, k - 1, d, device=x.device)
    # every sequence behind its k - 1 earlier inputs, so that a window is a run of rows
    at = torch.arange(total, device=x.device) + (seq + 1) * (k - 1)
    head = (starts[:-1] + torch.arange(count, device=x.device) * (k - 1))[:, None] + torch.arange(k - 1, device=x.device)
    padded = torch.empty(total + count * (k - 1), d, device=x.device)
    padded[at] = x
    padded[head.reshape(-1)] = initial.reshape(-1, d)
    window = at[:, None] - torch.arange(k - 1, -1, -1, device=x.device)     # [tokens, taps]
    c = (padded[window] * w.t()).sum(1) + bias
    y = torch.empty_like(c)
    y[rows] = F.silu(c)
    out = {"y": y.view(shape).to(dtype)}
    if case["ragged"]:
        tail = (starts[1:] + torch.arange(1, count + 1, device=x.device) * (k - 1))[:, None] - torch.arange(k - 1, 0, -1, device=x.device)
        out["state"] = padded[tail].to(dtype)
    if case["train"]:
        dc = dy.reshape(-1, d)[rows] * _silu_grad(c)
        dpadded = torch.zeros_like(padded)
        dpadded.index_add_(0, window.reshape(-1), (dc[:, None, :] * w.t()).reshape(-1, d))
        dx = torch.empty_like(x)
        dx[rows] = dpadded[at]
        out["d_x"] = dx.view(shape).to(dtype)
        out["d_weight"] = (dc[:, None, :] * padded[window]).sum(0).t().contiguous()
        out["d_bias"] = dc.sum(0)
        if s["initial"] is not None:
            out["d_initial"] = dpadded[head].to(dtype)
    return out


def _plain_conv_step(s):
    x, w, bias, state = _wide(s, "x", "weight", "bias", "state")
    slots = s["slots"].long()
    window = torch.cat([state[slots], x[:, None]], 1)                        # [batch, taps, channels]
    y = F.silu((window * w.t()).sum(1) + bias).to(s["x"].dtype)
    s["state_out"][slots] = window[:, 1:].to(s["state"].dtype)
    return {"y": y, "state": s["state_out"]}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 0 with h_{-1} = 0, in log2(length) steps over the whole axis."""
    step = 1
    while step < a.shape[0]:
        b = torch.cat([b[:step], a[step:] * b[:-step] + b[step:]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_scan(s, case):
    u, delta, A, B, C, D, z, bias, initial, dy = _wide(s, "u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial", "dy")
    dtype, shape, d, n, groups = s["u"].dtype, u.shape, case["channels"], case["states"], case["groups"]
    rows, seq, starts = _order(s, case, u.device)
    per, total, count = d // groups, rows.numel(), starts.numel() - 1
    # tokens of all sequences one after another, in scan order; [tokens, groups, channels / groups, states]
    u, raw, z = (t.reshape(-1, groups, per)[rows] for t in (u, delta, z))
    B, C = (t.reshape(-1, groups, 1, n)[rows] for t in (B, C))
    A, D, bias = A.view(groups, per, n), D.view(groups, per), bias.view(groups, per)
    raw = raw + bias
    step = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    first = starts[:-1][starts[1:] > starts[:-1]]
    live = torch.nonzero(starts[1:] > starts[:-1]).flatten()
    last = starts[1:][live] - 1
    a = torch.exp(step[..., None] * A)
    b = (step * u)[..., None] * B
    if initial is not None:
        h0 = initial.view(count, groups, per, n)
        b[first] += a[first] * h0[live]
    cut = a.clone()
    cut[first] = 0.0
    # equal lengths: one sequence a column, so that the doubling runs over a single length
    lay = (lambda t: t) if s["offsets"] is not None else (
        lambda t: t.view(count, -1, *t.shape[1:]).transpose(0, 1))
    unlay = (lambda t: t) if s["offsets"] is not None else (
        lambda t: t.transpose(0, 1).reshape(total, *t.shape[2:]))
    h = unlay(_doubling(lay(cut), lay(b)))
    inner = (C * h).sum(-1) + D * u
    gate = F.silu(z)
    y = torch.empty(total, d, device=u.device)
    y[rows] = (inner * gate).view(total, d)
    out = {"y": y.view(shape).to(dtype)}
    if case["ragged"]:
        final = h0.clone()
        final[live] = h[last]
        out["state"] = final.view(count, d, n)
    if not case["train"]:
        return out
    dy = dy.reshape(-1, groups, per)[rows]
    dinner = dy * gate
    # g_t = C_t dinner_t + a_{t+1} g_{t+1}, from the last token of each sequence to its first
    after = torch.zeros_like(a)
    after[:-1] = cut[1:]
    g = unlay(_doubling(lay(after).flip(0), lay(C * dinner[..., None]).flip(0)).flip(0))
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[first] = 0.0 if initial is None else h0[live]
    q = g * a * before                                                       # d loss / d (step A)
    gb = (g * B).sum(-1)
    dstep = (q * A).sum(-1) + gb * u
    draw_ = dstep * torch.sigmoid(raw)

    def back(t, like):
        r = torch.empty(total, t[0].numel(), device=t.device)
        r[rows] = t.reshape(total, -1)
        return r.view(like.shape).to(like.dtype)

    out["d_u"] = back(gb * step + dinner * D, s["u"])
    out["d_delta"] = back(draw_, s["delta"])
    out["d_A"] = (q * step[..., None]).sum(0).view(d, n)
    out["d_B"] = back((g * (step * u)[..., None]).sum(2), s["B"])
    out["d_C"] = back((h * dinner[..., None]).sum(2), s["C"])
    out["d_D"] = (dinner * u).sum(0).view(d)
    out["d_z"] = back(dy * inner * _silu_grad(z), s["z"])
    out["d_delta_bias"] = draw_.sum(0).view(d)
    if initial is not None:
        dh0 = torch.zeros_like(h0)
        dh0[live] = a[first] * g[first]
        out["d_initial"] = dh0.view(count, d, n)
    return out


def _plain_scan_step(s):
    u, delta, A, B, C, D, z, bias, state = _wide(s, "u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")
    slots = s["slots"].long()
    raw = delta + bias
    step = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    h = torch.exp(step[..., None] * A) * state[slots] + (step * u)[..., None] * B[:, None, :]
    y = (((h * C[:, None, :]).sum(-1) + D * u) * F.silu(z)).to(s["u"].dtype)
    s["state_out"][slots] = h
    return {"y": y, "state": s["state_out"]}


# ---- the definitions in 64 bits, token by token ---------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if not case["op"].endswith("step") and case["length"] > 20000:
        return None
    with torch.no_grad():
        v = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
        if case["op"] == "conv_step":
            return _exact_conv_step(s, v, case)
        if case["op"] == "scan_step":
            return _exact_scan_step(s, v, case)
        return _exact_conv(s, v, case) if case["op"] == "conv" else _exact_scan(s, v, case)


def _exact_conv_step(s, v, case):
    y, out = torch.zeros_like(v["x"]), v["state"].clone()
    at = s["slots"].long()
    y += v["bias"]
    for k in range(case["taps"]):
        y += v["weight"][:, k] * (v["x"] if k == case["taps"] - 1 else v["state"][at, k])
    for k in range(case["taps"] - 1):
        out[at, k] = v["x"] if k == case["taps"] - 2 else v["state"][at, k + 1]
    return {"y": y / (1.0 + torch.exp(-y)), "state": out}


def _exact_scan_step(s, v, case):
    at = s["slots"].long()
    step = torch.logaddexp(v["delta"] + v["delta_bias"], torch.zeros((), dtype=torch.float64, device=at.device))
    h = torch.exp(torch.einsum("bd,dn->bdn", step, v["A"])) * v["state"][at] + torch.einsum("bd,bn->bdn", step * v["u"], v["B"])
    y = torch.einsum("bdn,bn->bd", h, v["C"]) + v["D"] * v["u"]
    out = v["state"].clone()
    out[at] = h
    return {"y": y * v["z"] / (1.0 + torch.exp(-v["z"])), "state": out}


def _pieces(s, case):
    """(first row, end row) of each sequence in the flattened token axis."""
    if s["offsets"] is not None:
        return list(zip(s["cuts"][:-1], s["cuts"][1:]))
    return [(i * case["length"], (i + 1) * case["length"]) for i in range(case["batch"])]


def _exact_conv(s, v, case):
    d, k = case["channels"], case["taps"]
    x = v["x"].reshape(-1, d)
    y, dx = torch.empty_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(v["weight"]), torch.zeros_like(v["bias"])
    finals, dinitials = [], []
    for i, (lo, hi) in enumerate(_pieces(s, case)):
        seq = x[lo:hi].flip(0) if case["reverse"] else x[lo:hi]
        size = hi - lo
        seq = torch.cat([v["initial"][i] if "initial" in v else torch.zeros(k - 1, d, dtype=x.dtype, device=x.device), seq])
        finals.append(seq[size:])
        c = v["bias"].expand(size, d).clone()
        for j in range(k):
            c += v["weight"][:, j] * seq[j:j + size]
        sig = 1.0 / (1.0 + torch.exp(-c))
        y[lo:hi] = (c * sig).flip(0) if case["reverse"] else c * sig
        if case["train"]:
            dy = v["dy"].reshape(-1, d)[lo:hi]
            dc = (dy.flip(0) if case["reverse"] else dy) * (sig + c * sig * (1.0 - sig))
            dseq = torch.zeros_like(seq)
            for j in range(k):
                dseq[j:j + size] += v["weight"][:, j] * dc
                dw[:, j] += (dc * seq[j:j + size]).sum(0)
            db += dc.sum(0)
            dinitials.append(dseq[:k - 1])
            dx[lo:hi] = dseq[k - 1:].flip(0) if case["reverse"] else dseq[k - 1:]
    out = {"y": y.view(v["x"].shape)}
    if case["ragged"]:
        out["state"] = torch.stack(finals)
    if case["train"]:
        out.update(d_x=dx.view(v["x"].shape), d_weight=dw, d_bias=db)
        if "initial" in v:
            out["d_initial"] = torch.stack(dinitials)
    return out


def _exact_scan(s, v, case):
    d, n, groups, train = case["channels"], case["states"], case["groups"], case["train"]
    flat = {k: v[k].reshape(-1, d) for k in ("u", "delta", "z", "dy") if k in v}
    bc = {k: v[k].reshape(-1, groups, n) for k in ("B", "C")}
    A, bias, skip = v["A"], v["delta_bias"], v["D"]
    per = d // groups
    spread = lambda t: t.repeat_interleave(per, -2)                          # [.., groups, n] -> [.., d, n]
    pieces = _pieces(s, case)
    count = len(pieces)
    total = flat["u"].shape[0]
    step_all = torch.logaddexp(flat["delta"] + bias, torch.zeros((), dtype=A.dtype, device=A.device))
    # sequences side by side where they are equally long, one after another otherwise
    if s["offsets"] is None:
        lanes = [torch.arange(lo, hi, device=A.device) for lo, hi in pieces]
        plans = [(list(range(count)), torch.stack([r.flip(0) if case["reverse"] else r for r in lanes], 1))]
    else:
        plans = [([i], (torch.arange(lo, hi, device=A.device).flip(0) if case["reverse"]
                        else torch.arange(lo, hi, device=A.device))[:, None]) for i, (lo, hi) in enumerate(pieces)]
    h0 = v["initial"] if "initial" in v else torch.zeros(count, d, n, dtype=A.dtype, device=A.device)
    y = torch.empty_like(flat["u"])
    final, dh0 = h0.clone(), torch.zeros_like(h0)
    grads = {k: torch.zeros_like(t) for k, t in {**flat, **bc}.items()}
    dA, dD, dbias = torch.zeros_like(A), torch.zeros_like(skip), torch.zeros_like(bias)
    for ids, plan in plans:
        h, kept = h0[ids], []
        for rows in plan:                                                    # rows: one token of each sequence
            step, u = step_all[rows], flat["u"][rows]
            if train:
                kept.append(h)
            h = torch.exp(step[..., None] * A) * h + (step * u)[..., None] * spread(bc["B"][rows])
            y[rows] = (h * spread(bc["C"][rows])).sum(-1) + skip * u
        final[ids] = h
        if not train:
            continue
        g = torch.zeros_like(h)
        for rows, past in zip(reversed(plan), reversed(kept)):
            step, u, z, dy = step_all[rows], flat["u"][rows], flat["z"][rows], flat["dy"][rows]
            B = spread(bc["B"][rows])
            decay = torch.exp(step[..., None] * A)
            sig = 1.0 / (1.0 + torch.exp(-z))
            dinner = dy * z * sig
            grads["z"][rows] = dy * y[rows] * (sig + z * sig * (1.0 - sig))
            now = decay * past + (step * u)[..., None] * B
            g = g + spread(bc["C"][rows]) * dinner[..., None]
            grads["C"][rows] = (now * dinner[..., None]).view(-1, groups, per, n).sum(2)
            grads["B"][rows] = (g * (step * u)[..., None]).view(-1, groups, per, n).sum(2)
            gb = (g * B).sum(-1)
            g = g * decay
            q = g * past
            dA += (q * step[..., None]).sum(0)
            draw_ = ((q * A).sum(-1) + gb * u) / (1.0 + torch.exp(-flat["delta"][rows] - bias))
            grads["delta"][rows] = draw_
            dbias += draw_.sum(0)
            grads["u"][rows] = gb * step + dinner * skip
            dD += (dinner * u).sum(0)
        dh0[ids] = g
    z = flat["z"]
    out = {"y": (y * z / (1.0 + torch.exp(-z))).view(v["u"].shape)}
    if case["ragged"]:
        out["state"] = final
    if train:
        out.update(d_u=grads["u"].view(v["u"].shape), d_delta=grads["delta"].view(v["u"].shape), d_A=dA,
                   d_B=grads["B"].view(v["B"].shape), d_C=grads["C"].view(v["C"].shape), d_D=dD,
                   d_z=grads["z"].view(v["u"].shape), d_delta_bias=dbias)
        if "initial" in v:
            out["d_initial"] = dh0
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    size, d = (4 if case["type"] == "fp32" else 2), case["channels"]
    if case["op"] == "conv_step":
        k, b = case["taps"], case["batch"]
        return {"bytes": b * d * size * (2 + 2 * (k - 1)) + d * (k + 1) * 4, "flops": b * d * (2 * k + 4)}
    if case["op"] == "scan_step":
        n, b = case["states"], case["batch"]
        return {"bytes": b * d * (4 * size + 8 * n) + 2 * b * n * size + d * (n + 2) * 4, "flops": b * d * (7 * n + 10)}
    tokens = case["length"] * (1 if case["ragged"] else case["batch"])
    train = case["train"]
    states = case["batch"] if case["ragged"] else 0
    if case["op"] == "conv":
        k = case["taps"]
        moved = tokens * d * size * (4 if train else 2) + d * (k + 1) * 4 * (2 if train else 1)
        moved += states * (k - 1) * d * size * (3 if train else 2)
        return {"bytes": moved, "flops": tokens * d * ((6 * k + 12) if train else (2 * k + 4))}
    n, groups = case["states"], case["groups"]
    moved = tokens * size * ((8 * d + 4 * groups * n) if train else (4 * d + 2 * groups * n))
    moved += d * (n + 2) * 4 * (2 if train else 1) + states * d * n * 4 * (3 if train else 2)
    return {"bytes": moved, "flops": tokens * d * ((20 * n + 30) if train else (7 * n + 10))}
