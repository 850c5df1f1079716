"""Linear attention and the group norm as programs use them: shared heads, garbage in padding, several streams,
a first call inside a capture, tensors past 2^31 elements."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests.test_gpu_group_norm import normal as shifted
from tests.test_gpu_linear_attention import absolute, decays, near, normal, recurrence
from visionhope_b200.ssm_core import linear_attention, linear_attention_step
from visionhope_b200.utils.group_norm import group_norm, group_norm_rows

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_keys_and_values_shared_by_heads(dtype):
    """Expanded keys and values (a head stride of 0): the gradient sums over the heads that share them."""
    b, n, h, d = 2, 200, 4, 64
    q, k, v = normal(1, b, n, h, d, dtype=dtype), normal(2, b, n, 1, d, dtype=dtype), normal(3, b, n, 1, d, dtype=dtype)
    g, do = decays(h), normal(4, b, n, h, d, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = linear_attention(leaves[0], leaves[1].expand(b, n, h, d), leaves[2].expand(b, n, h, d), g)
    whole = (q, k.expand(b, n, h, d), v.expand(b, n, h, d))
    want = recurrence(*whole, g, d ** -0.5, None, False, do)
    size = recurrence(*absolute(*whole), g, d ** -0.5, None, False, do.abs())
    near(o, want[0], size[0], dtype, 5)
    got = torch.autograd.grad(o, leaves, do)
    near(got[0], want[2], size[2], dtype, 5)
    for x, w, s in ((got[1], want[3], size[3]), (got[2], want[4], size[4])):
        # each head's gradient is rounded to dtype before they are added (in dtype)
        s = s.sum(2, keepdim=True)
        near(x, w.sum(2, keepdim=True), s + 5 * w.abs().sum(2, keepdim=True), dtype, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reverse", [False, True])
def test_padding_may_hold_anything(dtype, reverse):
    """NaN in rows of no sequence, before, between chunk ends and behind: they reach nothing."""
    h, d, total, cuts = 2, 64, 900, [40, 300, 301, 750]
    q, k, v, do = (normal(i, total, h, d, dtype=dtype) for i in range(4))
    offsets, g = torch.tensor(cuts, device="cuda"), decays(h)
    clean = [t.clone().requires_grad_() for t in (q, k, v)]
    o, s = linear_attention(*clean, g, seq_offsets=offsets, return_final_state=True, reverse=reverse)
    grads = torch.autograd.grad(o, clean, do)
    for t in (q, k, v, do):
        t[:cuts[0]] = float("nan")
        t[cuts[-1]:] = float("nan")
    dirty = [t.clone().requires_grad_() for t in (q, k, v)]
    o2, s2 = linear_attention(*dirty, g, seq_offsets=offsets, return_final_state=True, reverse=reverse)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(o2, dirty, do)))


def test_calls_on_several_streams_at_once():
    """Calls of different shapes that share the SMs and their tensor memory."""
    shapes = [(4, 1000, 8, 64, 64), (2, 1000, 4, 128, 128), (8, 600, 4, 64, 128), (1, 3000, 2, 128, 64)]
    calls = []
    for i, (b, n, h, dk, dv) in enumerate(shapes):
        calls.append([normal(10 * i + j, b, n, h, d, dtype=torch.bfloat16) for j, d in enumerate((dk, dk, dv))] + [decays(h)])
    want = [linear_attention(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = [[] for _ in calls]
        for rep in range(4):
            for s, c, out in zip(streams, calls, got):
                with torch.cuda.stream(s):
                    out.append(linear_attention(*c))
        torch.cuda.synchronize()
        for w, out in zip(want, got):
            assert all(torch.equal(w, o) for o in out)


_FIRST = """
import torch
from visionhope_b200.ssm_core import linear_attention, linear_attention_step
from visionhope_b200.utils.group_norm import group_norm, group_norm_rows
torch.manual_seed(0)
q, k, v = (torch.randn(2, 700, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(3))
x = torch.randn(2, 64, 80, 80, device="cuda").contiguous(memory_format=torch.channels_last)
g = torch.full((2,), -0.1, device="cuda")
state = torch.zeros(2, 2, 64, 64, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    o, s = linear_attention(q, k, v, g, return_final_state=True)
    o1 = linear_attention(q.float(), k.float(), v.float(), g)
    y = group_norm(x, 8, activation="gelu")
    r = group_norm_rows(o.flatten(-2), 2)
    t = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
graph.replay()
w, ws = linear_attention(q, k, v, g, return_final_state=True)
assert torch.equal(o, w) and torch.equal(s, ws) and torch.equal(y, group_norm(x, 8, activation="gelu"))
assert torch.equal(r, group_norm_rows(w.flatten(-2), 2)) and torch.equal(o1, linear_attention(q.float(), k.float(), v.float(), g))
print("captured")
"""


def test_first_call_of_a_process_is_captured():
    """No set-up of the library has to come before a capture."""
    r = subprocess.run([sys.executable, "-c", _FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_past_2_to_the_31_elements(dtype):
    """The last tokens of rows whose elements need 64-bit offsets; the decays forget all but a few tokens."""
    heads, d = 16, 128
    n = 2 ** 31 // (3 * heads * d) + 1500
    rows = torch.empty(1, n, 3 * heads * d, device="cuda", dtype=dtype)
    for a in range(0, n, 65536):
        rows[:, a:a + 65536] = normal(a, 1, min(65536, n - a), 3 * heads * d, dtype=dtype)
    q, k, v = (t.view(1, n, heads, d) for t in rows.split(heads * d, dim=-1))
    g = torch.full((heads,), -1.0, device="cuda")
    o, s = linear_attention(q, k, v, g, return_final_state=True)
    tail = [t[:, -1600:] for t in (q, k, v)]
    want, end = recurrence(*tail, g, d ** -0.5, None)
    size, send = recurrence(*absolute(*tail), g, d ** -0.5, None)
    near(o[:, -1400:], want[:, -1400:], size[:, -1400:], dtype, 4)  # exp(-200) of what came before
    near(s, end, send, dtype, 4, operand=2 ** -22)


def test_images_past_2_to_the_31_elements():
    c, h, w = 64, 4100, 8200
    x = torch.empty(1, h, w, c, device="cuda", dtype=torch.bfloat16)
    total, square = torch.zeros(4, dtype=torch.float64, device="cuda"), torch.zeros(4, dtype=torch.float64, device="cuda")
    for a in range(0, h, 100):
        x[0, a:a + 100] = shifted(a, min(100, h - a), w, c, dtype=torch.bfloat16, scale=2.0, shift=0.5)
        part = x[0, a:a + 100].double().view(-1, 4, 16)
        total, square = total + part.sum((0, 2)), square + part.square().sum((0, 2))
    m = h * w * 16
    mean = total / m
    rstd = 1 / (square / m - mean * mean + 1e-5).sqrt()
    y = group_norm(x.permute(0, 3, 1, 2), 4).permute(0, 2, 3, 1)
    for part in (slice(0, 2), slice(h - 2, h)):
        want = ((x[0, part].double().view(-1, 4, 16) - mean.view(1, 4, 1)) * rstd.view(1, 4, 1)).view(2, w, c)
        # half a step of bf16, and sums of 2^29 values in fp32 parts, good to 2^-16 of the deviation
        assert bool(((y[0, part].double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -14).all())


def test_norm_of_unusual_rows():
    """Rows with a stride of 0, of one row, and of more than two axes with a gap between them."""
    row = normal(1, 1, 64)
    assert torch.equal(group_norm_rows(row.expand(5, 64), 4), group_norm_rows(row, 4).expand(5, 64))
    x = normal(2, 3, 7, 200, dtype=torch.bfloat16)[:, :, 100:164]
    assert torch.equal(group_norm_rows(x, 4), group_norm_rows(x.contiguous(), 4))
    t = normal(3, 64, 9).t()  # channels not adjacent
    assert torch.equal(group_norm_rows(t, 4), group_norm_rows(t.contiguous(), 4))


def test_step_takes_one_state_per_stream_in_any_order():
    """Steps with and without an index agree, and a stream skipped twice keeps its state."""
    q, k, v = (normal(i, 3, 2, 64, dtype=torch.bfloat16) for i in range(3))
    g, state = decays(2), normal(5, 3, 2, 64, 64)
    a, b = state.clone(), state.clone()
    oa = linear_attention_step(q, k, v, g, a)
    order = torch.tensor([2, 0, 1], device="cuda")
    ob = linear_attention_step(q[order], k[order], v[order], g, b, slots=order)
    assert torch.equal(oa[order], ob) and torch.equal(a, b)
    c = state.clone()
    linear_attention_step(q, k, v, g, c, slots=torch.tensor([-1, 5, -1], device="cuda"))
    assert torch.equal(c, state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 3000, 1, 64, 64), (1, 20000, 2, 64, 64), (1, 2500, 2, 128, 128)])
@pytest.mark.parametrize("reverse", [False, True])
def test_values_that_are_not_finite_in_segments(dtype, shape, reverse):
    """Where a sequence is cut into segments, tokens before an infinite value keep their bits outside its chunk."""
    b, n, h, dk, dv = shape
    q, k, v = (normal(i, b, n, h, d, dtype=dtype) for i, d in enumerate((dk, dk, dv)))
    g, at = decays(h), 1700
    clean = linear_attention(q, k, v, g, reverse=reverse)
    v[0, at, 0, 3] = float("inf")
    o = linear_attention(q, k, v, g, reverse=reverse)
    before = slice(at + 129, n) if reverse else slice(0, at - 128)
    after = slice(0, at + 1) if reverse else slice(at, n)
    assert torch.equal(o[:, before], clean[:, before]) and torch.equal(o[:, :, 1:], clean[:, :, 1:])
    others = torch.arange(dv, device="cuda") != 3
    chunk = slice(at + 1, at + 129) if reverse else slice(at - 128, at)
    near(o[:, chunk], clean[:, chunk].double(), clean[:, chunk].double().abs() + 30, dtype, 4, operand=2 ** -8 if dtype != torch.float32 else None)
    assert torch.isfinite(o[:, after, 0][..., others]).all() and not torch.isfinite(o[0, at, 0, 3])
