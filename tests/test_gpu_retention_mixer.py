"""The layer on linear attention and the gated group norm: whole, packed and cached use against its formula."""
import copy

import pytest
import torch

from tests.test_gpu_group_norm import formula
from visionhope_b200.retention_mixer import RetentionMixer
from visionhope_b200.ssm_mixer import image_rows

pytestmark = pytest.mark.gpu


def plain(m, x, reverse=False):
    """The layer in fp64 on [B, L, dim], differentiable."""
    h, dk, dv = m.heads, m.key_dim, m.value_dim
    q, k, v, gate = (x @ m.in_proj.weight.T).split((h * dk, h * dk, h * dv, h * dv), dim=-1)
    q, k, v = q.unflatten(-1, (h, dk)), k.unflatten(-1, (h, dk)), v.unflatten(-1, (h, dv))
    at = torch.arange(x.shape[1], device=x.device)
    ahead = at[None, :] - at[:, None] if reverse else at[:, None] - at[None, :]
    decay = torch.where(ahead >= 0, torch.exp(m.log_decay.double()[:, None, None] * ahead.clamp(min=0)), 0.0)
    o = torch.einsum("bihd,bjhd,hij,bjhe->bihe", q, k, decay, v) * dk ** -0.5
    flat = formula(o.flatten(-2).flatten(0, 1), h, m.norm_weight, m.norm_bias, m.eps, None, gate.flatten(0, 1))
    return flat.view(*x.shape[:2], -1) @ m.out_proj.weight.T


def layer(dim=64, seed=0, **kw):
    torch.manual_seed(seed)
    m = RetentionMixer(dim, **kw).cuda()
    with torch.no_grad():
        m.norm_weight.uniform_(0.5, 1.5)
        m.norm_bias.uniform_(-0.5, 0.5)
    return m


@pytest.mark.parametrize("dim,heads,key_dim,expand", [(64, 4, None, 2), (96, 3, 20, 1), (128, 2, 128, 2), (64, 1, 64, 2)])
@pytest.mark.parametrize("reverse", [False, True])
def test_layer_and_gradients(dim, heads, key_dim, expand, reverse):
    m = layer(dim, heads=heads, key_dim=key_dim, expand=expand)
    x = image_rows(torch.randn(2, dim, 9, 14, device="cuda").contiguous(memory_format=torch.channels_last)).requires_grad_()
    wide = copy.deepcopy(m).double()
    y, want = m(x, reverse=reverse), plain(wide, x.detach().double().requires_grad_(), reverse)
    assert torch.allclose(y.double(), want, atol=2e-4, rtol=1e-4)
    xd = x.detach().double().requires_grad_()
    dy = torch.randn_like(y)
    names = [n for n, _ in m.named_parameters()]
    got = torch.autograd.grad(y, [x, *m.parameters()], dy)
    exact = torch.autograd.grad(plain(wide, xd, reverse), [xd, *wide.parameters()], dy.double())
    for n, g, w in zip(["x", *names], got, exact):
        assert float((g.double() - w).norm() / w.norm()) < 1e-4, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_and_tokens(dtype):
    """Ragged prompts, packed, then tokens of some of the streams: as each stream's whole sequence."""
    m = layer(64, heads=4).to(dtype)
    m.log_decay = m.log_decay.float()
    lengths, more = [30, 1, 0, 77], 6
    total = sum(lengths)
    full = [torch.randn(n + more, 64, device="cuda").to(dtype) for n in lengths]
    packed = torch.cat([f[:n] for f, n in zip(full, lengths)])
    offsets = torch.tensor([0, 30, 31, 31, 108], device="cuda")
    y, state = m.prefill(packed, seq_offsets=offsets)
    cache = m.empty_cache(6)
    slots = torch.tensor([5, 0, 3, 2], device="cuda")
    cache[slots] = state
    outs = [[], [], [], []]
    for t in range(more):
        z = m.step(torch.stack([f[n + t] for f, n in zip(full, lengths)]), cache, slots=slots)
        for o, row in zip(outs, z):
            o.append(row)
    assert not cache[1].any() and not cache[4].any() and y.shape == (total, 64)
    tol = dict(atol=2e-4, rtol=1e-4) if dtype == torch.float32 else dict(atol=4e-2, rtol=4e-2)
    for i, f in enumerate(full):
        with torch.no_grad():
            whole = m(f[None])[0]
        a, e = int(offsets[i]), int(offsets[i + 1])
        assert torch.allclose(y[a:e], whole[:e - a], **tol)
        assert torch.allclose(torch.stack(outs[i]), whole[e - a:], **tol)
    # a prompt that continues a cache
    with torch.no_grad():
        y2, s2 = m.prefill(full[3][None, 77:], cache=state[3:4].contiguous())
    assert torch.allclose(y2[0], torch.stack(outs[3]), **tol) and torch.allclose(s2[0], cache[2], atol=1e-3, rtol=1e-2)


def test_autocast_training_step():
    m = layer(64, heads=2)
    x = torch.randn(2, 100, 64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
    assert y.dtype == torch.bfloat16
    y.float().square().mean().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in m.parameters())


def test_refusals():
    for kw in (dict(dim=64, heads=3), dict(dim=0), dict(dim=512, heads=2), dict(dim=64, windows=(0.5, 2.0)), dict(dim=64, windows=(8.0, 2.0)),
               dict(dim=256, heads=1, key_dim=64)):
        with pytest.raises(ValueError):
            RetentionMixer(**kw)
