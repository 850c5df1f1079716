"""The selective state space operators in plain PyTorch, token by token: the oracle of
``visionhope_b200.ssm_core``.  Run it in float64; autograd gives the gradients.

``offsets`` (a list) splits packed ``[tokens, channels]`` rows into sequences; without it the rows are
``[batch, length, channels]``."""
import torch


def _split(rows, offsets):
    if offsets is None:
        return list(rows)
    return [rows[a:b] for a, b in zip(offsets[:-1], offsets[1:])]


def _join(parts, offsets):
    return torch.stack(parts) if offsets is None else torch.cat(parts)


def short_conv(x, weight, bias=None, *, activation=None, initial_state=None, offsets=None, reverse=False):
    """(y, final_state) of the causal convolution."""
    d, k = weight.shape
    ys, finals = [], []
    for i, seq in enumerate(_split(x, offsets)):
        seq = seq.flip(0) if reverse else seq
        head = x.new_zeros(k - 1, d) if initial_state is None else initial_state[i]
        full = torch.cat([head, seq])
        out = sum(weight[:, j] * full[j:j + len(seq)] for j in range(k))
        if bias is not None:
            out = out + bias
        if activation == "silu":
            out = out * torch.sigmoid(out)
        ys.append(out.flip(0) if reverse else out)
        finals.append(full[len(seq):])
    return _join(ys, offsets), torch.stack(finals)


def ssm_scan(u, delta, A, B, C, D=None, *, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
             offsets=None, reverse=False):
    """(y, final_state) of the selective scan; B, C: [..., groups, states] or [..., states]."""
    d, n = A.shape
    if B.dim() == u.dim():
        B, C = B.unsqueeze(-2), C.unsqueeze(-2)
    per = d // B.shape[-2]
    s = delta if delta_bias is None else delta + delta_bias
    if delta_softplus:
        s = torch.logaddexp(s, torch.zeros((), dtype=s.dtype))
    B, C = B.repeat_interleave(per, -2), C.repeat_interleave(per, -2)
    ys, finals = [], []
    for i, parts in enumerate(zip(*(_split(t, offsets) for t in (u, s, B, C)))):
        ui, si, bi, ci = (p.flip(0) if reverse else p for p in parts)
        h = u.new_zeros(d, n) if initial_state is None else initial_state[i]
        out = []
        for t in range(len(ui)):
            h = torch.exp(si[t, :, None] * A) * h + (si[t] * ui[t])[:, None] * bi[t]
            out.append((h * ci[t]).sum(-1))
        out = torch.stack(out) if out else ui.new_zeros(0, d)
        ys.append(out.flip(0) if reverse else out)
        finals.append(h)
    y = _join(ys, offsets)
    if D is not None:
        y = y + D * u
    if z is not None:
        y = y * z * torch.sigmoid(z)
    return y, torch.stack(finals)
