"""The token-row mixer (visionhope_b200.ssm_mixer): its composition against the float64 oracle,
prompts then single tokens against the whole sequence, packed prompts against separate ones, image
rows read both ways, and a training step.

fp32 bars: the fp32 GEMMs' rounding (inner products of up to 128 terms of size 1: 128 * 2^-24 =
8e-6 of the terms' norm) passes through the scan's gate and the output projection: 1e-4 of the
largest output."""
import pytest
import torch

from oracle import ssm as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")


def _mixer(seed=0, **kw):
    from visionhope_b200.ssm_mixer import SelectiveMixer

    torch.manual_seed(seed)
    return SelectiveMixer(kw.pop("dim", 64), **kw).to(DEV)


def _oracle(m, x, offsets=None, reverse=False):
    """The mixer in float64 on the CPU."""
    p = {k: v.detach().double().cpu() for k, v in m.state_dict().items()}
    value, gate = (x.double().cpu() @ p["in_proj.weight"].T).chunk(2, dim=-1)
    value, _ = oracle.short_conv(value, p["conv_weight"], p["conv_bias"], activation="silu", offsets=offsets, reverse=reverse)
    step, b, c = (value @ p["x_proj.weight"].T).split((m.step_rank,) + (m.groups * m.states,) * 2, dim=-1)
    b, c = (t.unflatten(-1, (m.groups, m.states)) for t in (b, c))
    y, _ = oracle.ssm_scan(value, step @ p["step_proj.weight"].T, -p["rate_log"].exp(), b, c, p["skip"], z=gate,
                           delta_bias=p["step_bias"], delta_softplus=True, offsets=offsets, reverse=reverse)
    return y @ p["out_proj.weight"].T


def _close(a, e, bar):
    a, e = a.detach().double().cpu(), e.detach().double().cpu()
    assert a.shape == e.shape
    assert float((a - e).abs().max()) <= bar * float(e.abs().max())


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("kw", [dict(), dict(states=8, taps=3, groups=2), dict(dim=36, expand=1)])
def test_mixer_against_oracle(kw, reverse):
    m = _mixer(**kw)
    x = torch.randn(2, 45, m.dim, device=DEV)
    with torch.no_grad():
        _close(m(x, reverse=reverse), _oracle(m, x, reverse=reverse), 1e-4)


def test_packed_prompts_then_tokens_follow_the_sequences():
    """Three prompts of 0, 1 and 30 tokens as one packed batch, then six tokens each through
    the cache, in any slot order: every output is the whole sequence's."""
    m = _mixer(1)
    lens, more = [0, 1, 30], 6
    seqs = [torch.randn(n + more, m.dim, device=DEV) for n in lens]
    offsets = torch.tensor([0, 0, 1, 31], device=DEV)
    with torch.no_grad():
        whole = [m(s[None])[0] for s in seqs]
        y, cache = m.prefill(torch.cat([s[:n] for s, n in zip(seqs, lens)]), seq_offsets=offsets)
        scale = max(float(w.abs().max()) for w in whole)
        assert float((y - torch.cat([w[:n] for w, n in zip(whole, lens)])).abs().max()) <= 1e-4 * scale
        order = torch.tensor([2, 0, 1], device=DEV)
        for t in range(more):
            tok = torch.stack([seqs[i][lens[i] + t] for i in order.tolist()])
            out = m.step(tok, cache, slots=order)
            for row, i in enumerate(order.tolist()):
                assert float((out[row] - whole[i][lens[i] + t]).abs().max()) <= 1e-4 * scale
        # a second prompt on top of a cache, and a stream that starts from nothing
        y2, again = m.prefill(seqs[2][None, :20])
        y3, _ = m.prefill(seqs[2][None, 20:], cache=again)
        _close(y3[0], whole[2][20:], 1e-4)
        fresh = m.empty_cache(1)
        for t in range(4):
            _close(m.step(seqs[2][None, t], fresh)[0], whole[2][t], 1e-3)


def test_image_rows_train_under_autocast():
    """Channels-last image tokens, read forward and backward, bf16 autocast: every parameter gets
    a finite gradient and a few steps of descent lower the loss."""
    from visionhope_b200.ssm_mixer import image_rows

    m = _mixer(2)
    x = torch.randn(2, m.dim, 14, 14, device=DEV).contiguous(memory_format=torch.channels_last)
    rows = image_rows(x)
    assert rows.data_ptr() == x.data_ptr() and rows.shape == (2, 196, m.dim)
    target = torch.randn(2, 196, m.dim, device=DEV)
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    losses = []
    for _ in range(8):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(rows) + m(rows, reverse=True)
        loss = (y.float() - target).square().mean()
        loss.backward()
        for name, p in m.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all(), name
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0]


def test_step_replays_in_a_cuda_graph():
    """A captured step, replayed on new tokens, advances the cache as direct calls do."""
    m = _mixer(3)
    direct, captured = m.empty_cache(2), m.empty_cache(2)
    token = torch.randn(2, m.dim, device=DEV)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(token, m.empty_cache(2))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.step(token, captured)
        captured.conv.zero_()
        captured.scan.zero_()
        for _ in range(3):
            token.normal_()
            graph.replay()
            assert torch.equal(out, m.step(token, direct))
    assert torch.equal(captured.scan, direct.scan) and torch.equal(captured.conv, direct.conv)


def test_sequences_replay_in_a_cuda_graph():
    """A captured forward over sequences (several dependent launches) gives the direct call's rows."""
    m = _mixer(4)
    rows = torch.randn(2, 700, m.dim, device=DEV)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(rows)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(rows)
        for _ in range(3):
            rows.normal_()
            graph.replay()
            assert torch.equal(out, m(rows))


def test_mixer_refuses():
    from visionhope_b200.ssm_mixer import SelectiveMixer

    with pytest.raises(ValueError):
        SelectiveMixer(0)
    with pytest.raises(ValueError):
        SelectiveMixer(10, groups=3)
    m = _mixer(states=12)
    with pytest.raises(ValueError, match="states"):
        m(torch.randn(1, 4, 64, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA"):
        SelectiveMixer(16)(torch.randn(1, 4, 16))
