"""Linear attention with a decay for each head against the recurrence in 64 bits, token by token."""
import math

import pytest
import torch

from visionhope_b200.ssm_core import linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# What the operands of the matrix products are rounded to, summed over the products that a term passes:
# bf16 scores or states once (2^-8, and 2^-16 of second order); fp16 as two planes (2^-17) with 2^-16
# dropped of each of two products; fp32 as three with 2^-24 dropped of each.
OPERAND = {torch.bfloat16: 2 ** -8 + 2 ** -15, torch.float16: 2 ** -14, torch.float32: 2 ** -22}


def decays(heads, device="cuda"):
    return torch.log1p(-torch.exp2(-1.0 - 6.0 * torch.arange(heads, device=device, dtype=torch.float32) / max(1, heads - 1)))


def normal(seed, *shape, dtype=torch.float32, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def recurrence(q, k, v, g, scale, initial, reverse=False, do=None, dfinal=None):
    """One batch of equally long sequences in fp64: o, final state and, with ``do``, the gradients."""
    q, k, v = (t.double() for t in (q, k, v))
    lam = torch.exp(g.double())[:, None, None]
    b, n, h, dk = q.shape
    s = torch.zeros(b, h, dk, v.shape[-1], dtype=torch.float64, device=q.device) if initial is None else initial.double()
    order = range(n - 1, -1, -1) if reverse else range(n)
    o, dq = torch.zeros_like(v), torch.zeros_like(q)
    for t in order:
        s = lam * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * (q[:, t, :, :, None] * s).sum(-2)
        if do is not None:
            dq[:, t] = scale * (s * do[:, t, :, None, :].double()).sum(-1)
    if do is None:
        return o, s
    ds = torch.zeros_like(s) if dfinal is None else dfinal.double()
    dk_, dv_ = torch.zeros_like(k), torch.zeros_like(v)
    for t in reversed(order):
        ds = ds + scale * q[:, t, :, :, None] * do[:, t, :, None, :].double()
        dk_[:, t] = (ds * v[:, t, :, None, :]).sum(-1)
        dv_[:, t] = (ds * k[:, t, :, :, None]).sum(-2)
        ds = lam * ds
    return o, s, dq, dk_, dv_, ds


def absolute(*tensors):
    return [None if t is None else t.double().abs() for t in tensors]


def near(got, want, size, dtype, chunks, operand=None):
    """|got - want| within the rounding of the result, of the operands (on ``size``, the same sum of absolute
    values) and of the fp32 sums: some 24 additions a chunk to a state and 150 to an output, each off by at
    most 2^-23 of the sum."""
    operand = OPERAND[dtype] if operand is None else operand
    out = torch.finfo(got.dtype).eps / 2
    tol = out * want.abs() + (operand + (24 * chunks + 150) * 2 ** -23) * 1.01 * size + 1e-30
    if got.dtype == torch.float16:
        tol = tol + 2 ** -25  # below the smallest normal number the step is 2^-24
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    bad = (off > tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} of the tolerance"


SHAPES = [(1, 1, 1, 64, 64), (2, 2, 3, 16, 16), (2, 63, 2, 64, 64), (1, 64, 2, 64, 128), (3, 65, 2, 32, 48), (2, 200, 2, 128, 128),
          (1, 129, 3, 100, 60), (2, 130, 2, 7, 5), (1, 1, 2, 1, 1), (2, 128, 1, 72, 33), (1, 1500, 2, 64, 64), (2, 1025, 1, 128, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_sequences(dtype, shape, reverse):
    """Outputs, final states and gradients, with and without states, from strided rows of one projection."""
    b, n, h, dk, dv = shape
    rows = normal(1, b, n, h * (2 * dk + dv) + 3, dtype=dtype)
    q = rows[..., :h * dk].view(b, n, h, dk)
    k = rows[..., h * dk:2 * h * dk].view(b, n, h, dk)
    v = rows[..., 2 * h * dk:h * (2 * dk + dv)].view(b, n, h, dv)
    g, scale, chunks = decays(h), dk ** -0.5, n // 64 + 2
    for with_states in (False, True):
        initial = normal(2, b, h, dk, dv) if with_states else None
        do = normal(3, b, n, h, dv, dtype=dtype)
        dfinal = normal(4, b, h, dk, dv) if with_states else None
        want = recurrence(q, k, v, g, scale, initial, reverse, do, dfinal)
        aq, ak, av, ai, ado, adf = absolute(q, k, v, initial, do, dfinal)
        size = recurrence(aq, ak, av, g, scale, ai, reverse, ado, adf)
        leaves = [t.detach().requires_grad_() if t is not None else None for t in (q, k, v, initial)]  # strides as they are
        plain, final = linear_attention(q, k, v, g, initial_state=initial, return_final_state=True, reverse=reverse)
        near(plain, want[0], size[0], dtype, chunks)
        near(final, want[1], size[1], dtype, chunks, operand=2 ** -15 if dtype == torch.float16 else 2 ** -22)
        o, final2 = linear_attention(*leaves[:3], g, initial_state=leaves[3], return_final_state=True, reverse=reverse)
        assert torch.equal(o, plain) and torch.equal(final2, final)
        outs, grads = ([o, final2], [do, dfinal]) if with_states else ([o], [do])
        live = [t for t in leaves if t is not None]
        got = torch.autograd.grad(outs, live, grads)
        for x, w, s in zip(got, want[2:], size[2:]):
            exact = x.dtype == torch.float32 and dtype != torch.float32
            near(x, w, s, dtype, chunks, operand=2 ** -15 if exact else None)


ALIGNED = [(1, 128, 1, 64, 64), (2, 129, 3, 64, 64), (1, 200, 2, 128, 128), (2, 255, 2, 64, 128), (1, 384, 2, 128, 64), (3, 777, 2, 64, 64),
           (1, 300, 2, 72, 104), (2, 640, 1, 16, 8), (1, 5000, 2, 128, 128), (1, 4099, 1, 64, 64), (40, 257, 4, 64, 64), (2, 100, 2, 64, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ALIGNED)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("with_states", [False, True])
def test_aligned_rows(dtype, shape, reverse, with_states):
    """As above from rows that start on 16 bytes, where wide copies and tiles are taken."""
    b, n, h, dk, dv = shape
    rows = normal(1, b, n, h * (2 * dk + dv), dtype=dtype)
    q, k, v = rows.split((h * dk, h * dk, h * dv), dim=-1)
    q, k, v = q.view(b, n, h, dk), k.view(b, n, h, dk), v.view(b, n, h, dv)
    g, scale, chunks = decays(h), dk ** -0.5, n // 64 + 2
    initial = normal(2, b, h, dk, dv) if with_states else None
    do = normal(3, b, n, h, dv, dtype=dtype)
    dfinal = normal(4, b, h, dk, dv) if with_states else None
    want = recurrence(q, k, v, g, scale, initial, reverse, do, dfinal)
    size = recurrence(*absolute(q, k, v), g, scale, *absolute(initial), reverse, *absolute(do, dfinal))
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (q, k, v, initial)]
    got = linear_attention(*leaves[:3], g, initial_state=leaves[3], return_final_state=with_states, reverse=reverse)
    o = got[0] if with_states else got
    near(o, want[0], size[0], dtype, chunks)
    if with_states:
        near(got[1], want[1], size[1], dtype, chunks, operand=2 ** -15 if dtype == torch.float16 else 2 ** -22)
    live = [t for t in leaves if t is not None]
    grads = torch.autograd.grad([o, got[1]] if with_states else [o], live, [do, dfinal] if with_states else [do])
    for x, w, s in zip(grads, want[2:], size[2:]):
        near(x, w, s, dtype, chunks, operand=2 ** -15 if x.dtype == torch.float32 and dtype != torch.float32 else None)


def test_default_scale_and_no_state():
    q, k, v = (normal(i, 1, 70, 2, 64, dtype=torch.bfloat16) for i in range(3))
    g = decays(2)
    assert torch.equal(linear_attention(q, k, v, g), linear_attention(q, k, v, g, scale=0.125))
    o, s = linear_attention(q, k, v, g, initial_state=torch.zeros(1, 2, 64, 64, device="cuda"), return_final_state=True)
    assert torch.equal(o, linear_attention(q, k, v, g)) and s.shape == (1, 2, 64, 64)


CUTS = [[0, 0, 5, 6, 6, 70, 300, 300, 1000, 1000], [3, 3, 200, 201, 900], [0, 1000], [0, 0], [500, 500, 500]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cuts", CUTS)
@pytest.mark.parametrize("reverse", [False, True])
def test_packed(dtype, cuts, reverse):
    """Packed sequences are their sequences one by one, and rows of none get zeros; the offsets may be int64."""
    h, dk, dv, total = 2, 64, 72, 1000
    q, k, v = (normal(i, total, h, d, dtype=dtype) for i, d in enumerate((dk, dk, dv)))
    n, g = len(cuts) - 1, decays(2)
    initial, do, dfinal = normal(5, n, h, dk, dv), normal(6, total, h, dv, dtype=dtype), normal(7, n, h, dk, dv)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, initial)]
    for kind in (torch.int32, torch.int64):
        offsets = torch.tensor(cuts, dtype=kind, device="cuda")
        o, final = linear_attention(*leaves[:3], g, initial_state=leaves[3], return_final_state=True, seq_offsets=offsets,
                                    reverse=reverse)
        got = torch.autograd.grad([o, final], leaves, [do, dfinal])
        for t in (o, *got[:3]):
            assert not t[:cuts[0]].any() and not t[cuts[-1]:].any()
        for i, (a, e) in enumerate(zip(cuts[:-1], cuts[1:])):
            one = [t[None, a:e] for t in (q, k, v)]
            want = recurrence(*one, g, dk ** -0.5, initial[i:i + 1], reverse, do[None, a:e], dfinal[i:i + 1])
            size = recurrence(*absolute(*one), g, dk ** -0.5, initial[i:i + 1].abs(), reverse, do[None, a:e].abs(), dfinal[i:i + 1].abs())
            have = (o[None, a:e], final[i:i + 1], *(t[None, a:e] for t in got[:3]), got[3][i:i + 1])
            for x, w, s in zip(have, want, size):
                if x.numel():
                    exact = x.dtype == torch.float32 and dtype != torch.float32
                    near(x, w, s, dtype, (e - a) // 64 + 2, operand=2 ** -15 if exact else None)


def test_offsets_outside_are_clamped():
    """Offsets past the tokens end at them, whatever their values."""
    q, k, v = (normal(i, 300, 2, 64, dtype=torch.bfloat16) for i in range(3))
    g = decays(2)
    want = linear_attention(q, k, v, g, seq_offsets=torch.tensor([0, 100, 300], device="cuda"))
    got = linear_attention(q, k, v, g, seq_offsets=torch.tensor([-5, 100, 1 << 40], device="cuda"))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_memory_and_none(dtype):
    """Decays of one (a plain sum), of nearly nothing and of nothing: minus infinity keeps a token's own term only."""
    g = torch.tensor([0.0, -60.0, -math.inf], device="cuda")
    b, n, h, dk, dv = 1, 700, 3, 32, 64
    q, k, v = (normal(i, b, n, h, d, dtype=dtype) for i, d in enumerate((dk, dk, dv)))
    initial = normal(9, b, h, dk, dv)
    want = recurrence(q, k, v, g, 1.0, initial)
    size = recurrence(*absolute(q, k, v), g, 1.0, initial.abs())
    o, s = linear_attention(q, k, v, g, scale=1.0, initial_state=initial, return_final_state=True)
    near(o, want[0], size[0], dtype, n // 64 + 2)
    near(s, want[1], size[1], dtype, n // 64 + 2, operand=2 ** -15 if dtype == torch.float16 else 2 ** -22)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("reverse", [False, True])
def test_values_that_are_not_finite_reach_later_tokens_only(dtype, name, bad, reverse):
    """An infinity or NaN in one token leaves the tokens before it, and other sequences, as they were."""
    h, d, total = 2, 64, 400
    cuts = [0, 150, 150, 290, 400]
    t = dict(q=normal(1, total, h, d, dtype=dtype), k=normal(2, total, h, d, dtype=dtype), v=normal(3, total, h, d, dtype=dtype))
    offsets, g = torch.tensor(cuts, device="cuda"), decays(2)
    clean, s0 = linear_attention(t["q"], t["k"], t["v"], g, seq_offsets=offsets, return_final_state=True, reverse=reverse)
    at = 200
    t[name][at, 1, 5] = bad
    o, s = linear_attention(t["q"], t["k"], t["v"], g, seq_offsets=offsets, return_final_state=True, reverse=reverse)
    free = torch.ones(total, dtype=torch.bool, device="cuda")
    if name == "q":
        free[at] = False
    elif reverse:
        free[150:at + 1] = False
    else:
        free[at:290] = False
    assert torch.equal(o[:, 0], clean[:, 0])
    # where a chunk is summed again, term by term, the order of the sums differs
    near(o[free][:, 1], clean[free][:, 1].double(), clean[free][:, 1].double().abs() + 30, dtype, 4, operand=2 ** -8 if dtype != torch.float32 else None)
    assert not torch.isfinite(o[at, 1]).all()
    keep = [0, 1, 3] if name != "q" else [0, 1, 2, 3]
    assert torch.equal(s[keep], s0[keep]) and torch.equal(s[:, 0], s0[:, 0])


def test_gradients_against_differences():
    """o is linear in q, in k and in v alone, and in the initial state: differences are exact up to rounding."""
    b, n, h, dk, dv = 2, 150, 2, 48, 40
    q, k, v = (normal(i, b, n, h, d) for i, d in ((0, dk), (1, dk), (2, dv)))
    initial = normal(3, b, h, dk, dv)
    g = decays(h)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, initial)]
    o, s = linear_attention(*leaves[:3], g, initial_state=leaves[3], return_final_state=True)
    wo, ws = normal(4, *o.shape), normal(5, *s.shape)
    grads = torch.autograd.grad([o, s], leaves, [wo, ws])

    def loss(*t):
        o, s = linear_attention(*t[:3], g, initial_state=t[3], return_final_state=True)
        return (o.double() * wo.double()).sum() + (s.double() * ws.double()).sum()

    for i in range(4):
        d = normal(10 + i, *leaves[i].shape)
        plus, minus = [t.detach() for t in leaves], [t.detach() for t in leaves]
        plus[i], minus[i] = plus[i] + d, minus[i] - d
        want = (loss(*plus) - loss(*minus)) / 2
        got = (grads[i].double() * d.double()).sum()
        # every element of the sums is off by some 2^-21 of values near 10, 30000 of them with either sign
        assert abs(float(got - want)) <= 0.02 + 1e-4 * abs(float(want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,slots,h,dk,dv", [(1, 1, 1, 64, 64), (5, 9, 3, 128, 128), (3, 3, 2, 40, 72), (2, 4, 2, 7, 5), (40, 64, 4, 64, 128), (1, 2, 1, 1, 1)])
def test_step(dtype, batch, slots, h, dk, dv):
    """One token: in place, into another buffer, with slots outside the cache skipped."""
    q, k, v = (normal(i, batch, h, d, dtype=dtype) for i, d in enumerate((dk, dk, dv)))
    state, g = normal(4, slots, h, dk, dv), decays(h)
    index = torch.randperm(slots, generator=torch.Generator().manual_seed(3))[:batch].cuda()
    want, end = recurrence(q[:, None], k[:, None], v[:, None], g, 0.3, state[index])
    size, send = recurrence(*absolute(q[:, None], k[:, None], v[:, None]), g, 0.3, state[index].abs())
    out = state.clone()
    o = linear_attention_step(q, k, v, g, out, scale=0.3, slots=index)
    near(o, want[:, 0], size[:, 0], dtype, 1, operand=0)
    near(out[index], end, send, dtype, 1, operand=0)
    rest = torch.ones(slots, dtype=torch.bool, device="cuda")
    rest[index] = False
    assert torch.equal(out[rest], state[rest])
    other = torch.full_like(state, 7.0)
    o2 = linear_attention_step(q, k, v, g, state, scale=0.3, slots=index.int(), state_out=other)
    assert torch.equal(o2, o) and torch.equal(other[index], out[index]) and bool((other[rest] == 7).all())
    # a state that does not start on 16 bytes
    raw = torch.empty(state.numel() + 1, device="cuda")
    odd = raw[1:].view_as(state).copy_(state)
    o3 = linear_attention_step(q, k, v, g, odd, scale=0.3, slots=index)
    near(o3, want[:, 0], size[:, 0], dtype, 1, operand=0)
    near(odd[index], end, send, dtype, 1, operand=0)
    # slots outside
    far = index.clone()
    far[0] = slots
    again = state.clone()
    o4 = linear_attention_step(q, k, v, g, again, scale=0.3, slots=far)
    assert not o4[0].any() and torch.equal(o4[1:], o[1:]) and torch.equal(again[index[0]], state[index[0]])


def test_steps_continue_a_sequence():
    """A prompt and then single tokens give what the whole sequence gives."""
    b, n, m, h, d = 2, 100, 20, 2, 64
    q, k, v = (normal(i, b, n + m, h, d) for i in range(3))
    g = decays(h)
    whole, end = linear_attention(q, k, v, g, return_final_state=True)
    o, state = linear_attention(q[:, :n], k[:, :n], v[:, :n], g, return_final_state=True)
    outs = [o] + [linear_attention_step(q[:, t], k[:, t], v[:, t], g, state)[:, None] for t in range(n, n + m)]
    assert torch.allclose(torch.cat(outs, 1), whole, rtol=1e-5, atol=2e-5) and torch.allclose(state, end, rtol=1e-5, atol=2e-5)


def test_two_calls_give_the_same_bits():
    q, k, v = (normal(i, 2, 3000, 2, 64, dtype=torch.bfloat16).requires_grad_() for i in range(3))
    do = normal(5, 2, 3000, 2, 64, dtype=torch.bfloat16)
    runs = []
    for _ in range(2):
        o = linear_attention(q, k, v, decays(2))
        runs.append((o, *torch.autograd.grad(o, (q, k, v), do)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_streams_and_graphs():
    """On a stream of the caller's, and captured: replays read the inputs as they are then."""
    q, k, v = (normal(i, 2, 500, 2, 64, dtype=torch.bfloat16) for i in range(3))
    g = decays(2)
    state = normal(6, 2, 2, 64, 64)
    want = linear_attention(q, k, v, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = linear_attention(q, k, v, g)
        s = state.clone()
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want)
    x, y, z = (t.clone() for t in (q, k, v))
    graph, s2 = torch.cuda.CUDAGraph(), state.clone()
    leaves = [t.requires_grad_() for t in (x, y, z)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(linear_attention(*leaves, g), leaves, torch.ones_like(v))
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        o2 = linear_attention(*leaves, g)
        grads = torch.autograd.grad(o2, leaves, torch.ones_like(v))
        with torch.no_grad():
            o3 = linear_attention_step(x[:, 0], y[:, 0], z[:, 0], g, s2)
    for seed in (20, 21):
        with torch.no_grad():
            for i, t in enumerate(leaves):
                t.copy_(normal(seed + i, *t.shape, dtype=t.dtype))
            s2.copy_(state)
        graph.replay()
        fresh = [t.detach().clone().requires_grad_() for t in leaves]
        w = linear_attention(*fresh, g)
        assert torch.equal(o2, w)
        assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(w, fresh, torch.ones_like(v))))
        s = state.clone()
        assert torch.equal(o3, linear_attention_step(fresh[0][:, 0].detach(), fresh[1][:, 0].detach(), fresh[2][:, 0].detach(), g, s))
        assert torch.equal(s2, s)


def test_no_wait_gave_up():
    """After everything above, none of the tensor-core kernels' bounded waits has run out."""
    from visionhope_b200 import _lib

    assert _lib.load().vh_tc_status(0) == 0


@pytest.mark.parametrize("shape", [(0, 5, 2, 64, 64), (2, 0, 2, 64, 64), (2, 5, 0, 64, 64)])
def test_nothing_to_do(shape):
    b, n, h, dk, dv = shape
    q, k, v = (torch.zeros(b, n, h, d, device="cuda", requires_grad=True) for d in (dk, dk, dv))
    initial = torch.ones(b, h, dk, dv, device="cuda", requires_grad=True)
    o, s = linear_attention(q, k, v, torch.zeros(h, device="cuda"), initial_state=initial, return_final_state=True)
    assert o.shape == (b, n, h, dv) and torch.equal(s, initial)
    got = torch.autograd.grad([o, s], [q, k, v, initial], [torch.ones_like(o), torch.full_like(s, 3.0)])
    assert [t.shape for t in got] == [t.shape for t in (q, k, v, initial)] and bool((got[3] == 3).all())


def test_only_one_gradient_arrives():
    """Through the final state alone, and through o alone."""
    q, k, v = (normal(i, 1, 90, 2, 32).requires_grad_() for i in range(3))
    g = decays(2)
    o, s = linear_attention(q, k, v, g, return_final_state=True)
    want = recurrence(q, k, v, g, 32 ** -0.5, None, False, torch.zeros_like(v), torch.ones_like(s))
    size = recurrence(*absolute(q, k, v), g, 32 ** -0.5, None, False, torch.zeros_like(v), torch.ones_like(s))
    got = torch.autograd.grad(s.sum(), (k, v), retain_graph=True)
    near(got[0], want[3], size[3], torch.float32, 3)
    near(got[1], want[4], size[4], torch.float32, 3)


def test_refusals():
    q = torch.zeros(2, 5, 2, 64, device="cuda", dtype=torch.bfloat16)
    g = torch.zeros(2, device="cuda")
    with pytest.raises(ValueError, match="k must have shape"):
        linear_attention(q, q[:, :4], q, g)
    with pytest.raises(ValueError, match="v must"):
        linear_attention(q, q, q[:, :4], g)
    with pytest.raises(ValueError, match="v must be"):
        linear_attention(q, q, q[0], g)
    with pytest.raises(TypeError, match="k must be"):
        linear_attention(q, q.float(), q, g)
    with pytest.raises(TypeError, match="unsupported dtype"):
        linear_attention(q.double(), q.double(), q.double(), g)
    with pytest.raises(ValueError, match="log_decay must have shape"):
        linear_attention(q, q, q, g[:1])
    with pytest.raises(ValueError, match="constant"):
        linear_attention(q, q, q, g.clone().requires_grad_())
    with pytest.raises(ValueError, match="initial_state must have shape"):
        linear_attention(q, q, q, g, initial_state=torch.zeros(2, 2, 64, 32, device="cuda"))
    with pytest.raises(TypeError, match="initial_state must be"):
        linear_attention(q, q, q, g, initial_state=torch.zeros(2, 2, 64, 64, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="q must be"):
        linear_attention(q[0], q[0], q[0], g)
    with pytest.raises(ValueError, match="q must be"):
        linear_attention(q, q, q, g, seq_offsets=torch.tensor([0, 5], device="cuda"))
    with pytest.raises(TypeError, match="seq_offsets"):
        linear_attention(q[0], q[0], q[0], g, seq_offsets=torch.tensor([0.0, 5.0], device="cuda"))
    wide = torch.zeros(1, 3, 2, 136, device="cuda")
    with pytest.raises(ValueError, match="dims of 1 to 128"):
        linear_attention(wide, wide, wide, g)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_attention(q.cpu(), q.cpu(), q.cpu(), g.cpu())
    state = torch.zeros(4, 2, 64, 64, device="cuda")
    one = q[:, 0]
    with pytest.raises(ValueError, match="state must have shape"):
        linear_attention_step(one, one, one, g, state[:, :1])
    with pytest.raises(ValueError, match="contiguous"):
        linear_attention_step(one, one, one, g, state.transpose(2, 3))
    with pytest.raises(ValueError, match="slots for"):
        linear_attention_step(one, one, one, g, state[:1])
    with pytest.raises(TypeError, match="state must be"):
        linear_attention_step(one, one, one, g, state.half())
    with pytest.raises(ValueError, match="slots must have shape"):
        linear_attention_step(one, one, one, g, state, slots=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="cache requires gradients"):
        linear_attention_step(one, one, one, g, state.clone().requires_grad_())
    y = linear_attention_step(one.float().requires_grad_(), one.float(), one.float(), g, state)
    with pytest.raises(RuntimeError, match="not differentiable"):
        y.sum().backward()
    x = torch.zeros(1, 5, 2, 64, device="cuda", requires_grad=True)
    d, = torch.autograd.grad(linear_attention(x, x, x, g).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)
