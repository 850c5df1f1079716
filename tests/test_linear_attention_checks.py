"""What the linear attention entry points answer without a GPU: the argument struct's layout, sizes and
refusals."""
import ctypes
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def _args(**kw):
    from visionhope_b200 import _lib

    keep = (ctypes.c_float * 64)()
    p = ctypes.addressof(keep)
    p += -p % 16
    a = _lib.VhLinearAttentionArgs(q=p, k=p, v=p, log_decay=p, o=p, length=128, scale=1.0, dtype=1, batch=2, heads=4, key_dim=64,
                                   value_dim=64, reverse=0)
    for n in ("q", "k", "v"):
        setattr(a, f"{n}_batch_stride", 128 * 256)
        setattr(a, f"{n}_token_stride", 256)
        setattr(a, f"{n}_head_stride", 64)
    for n, v in kw.items():
        setattr(a, n, v(p) if callable(v) else v)
    return a, p, keep


def _err():
    from visionhope_b200 import _lib

    return _lib.load().vh_last_error().decode()


def test_struct_layout(tmp_path):
    """The ctypes mirror and the packed form agree with the C header."""
    from visionhope_b200 import _lib
    from visionhope_b200.ssm_core import linear

    names = [n for n, _ in _lib.VhLinearAttentionArgs._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "vhope.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu\\n", offsetof(vh_linear_attention_args, {n}));\n' for n in names)
                   + 'printf("%zu\\n", sizeof(vh_linear_attention_args));\nreturn 0; }\n')
    exe = tmp_path / "o"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    want = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert want[:-1] == [getattr(_lib.VhLinearAttentionArgs, n).offset for n in names]
    assert want[-1] == ctypes.sizeof(_lib.VhLinearAttentionArgs) == linear._ARGS.size


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(log_decay=None), "null"), (dict(o=None), "null"), (dict(dtype=7), "dtype"),
    (dict(batch=0), "positive"), (dict(heads=-1), "positive"), (dict(heads=70000), "65535"), (dict(key_dim=0), "1 to 128"),
    (dict(key_dim=129), "1 to 128"), (dict(value_dim=256), "1 to 128"), (dict(length=-1), "negative"),
    (dict(length=1 << 31), "2^31"), (dict(q=lambda p: p + 1), "misaligned"), (dict(initial_state=lambda p: p + 2), "misaligned"),
    (dict(seq_offsets=lambda p: p + 2), "misaligned")])
def test_refused_arguments(change, text):
    from visionhope_b200 import _lib

    lib = _lib.load()
    a, p, keep = _args(**change)
    assert lib.vh_linear_attention_fwd(ctypes.byref(a), None, 0, None) < 0 and text in _err()
    if "o" not in change:
        assert lib.vh_linear_attention_bwd(ctypes.byref(a), p, None, p, p, p, None, None, 0, None) < 0 and text in _err()
    if not set(change) & {"length"}:
        assert lib.vh_linear_attention_step(ctypes.byref(a), p, p, None, 2, None) < 0 and text in _err()


def test_refused_workspaces_states_and_gradients():
    from visionhope_b200 import _lib

    lib = _lib.load()
    a, p, keep = _args(batch=1, length=100000)
    need = lib.vh_linear_attention_fwd_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.vh_linear_attention_fwd(ctypes.byref(a), None, need, None) < 0 and "workspace" in _err()
    assert lib.vh_linear_attention_fwd(ctypes.byref(a), p, need - 1, None) < 0 and "workspace" in _err()
    assert lib.vh_linear_attention_fwd(ctypes.byref(a), p + 4, need, None) == -5
    assert lib.vh_linear_attention_bwd_workspace_bytes(ctypes.byref(a)) >= need
    assert lib.vh_linear_attention_bwd(ctypes.byref(a), None, None, p, p, p, None, p, 1 << 40, None) < 0 and "null" in _err()
    assert lib.vh_linear_attention_bwd(ctypes.byref(a), p, None, p + 1, p, p, None, p, 1 << 40, None) == -5
    a, p, keep = _args()
    assert lib.vh_linear_attention_step(ctypes.byref(a), None, p, None, 4, None) < 0 and "state" in _err()
    assert lib.vh_linear_attention_step(ctypes.byref(a), p + 2, p, None, 4, None) == -5
    assert lib.vh_linear_attention_step(ctypes.byref(a), p, p, None, 1, None) < 0 and "slots" in _err()
    a.batch = 70000
    assert lib.vh_linear_attention_step(ctypes.byref(a), p, p, None, 70000, None) < 0 and "65535" in _err()
    assert lib.vh_linear_attention_fwd_workspace_bytes(None) == 0 and lib.vh_linear_attention_fwd(None, None, 0, None) < 0


@pytest.mark.parametrize("batch,length,packed", [(1, 0, False), (1, 1, False), (64, 784, False), (2, 16384, False), (24, 16384, True),
                                                 (5000, 20000, True), (1, (1 << 31) - 1, False)])
@pytest.mark.parametrize("heads,dk,dv", [(1, 1, 1), (4, 64, 64), (16, 128, 128), (3, 64, 128)])
def test_workspace_is_as_documented(batch, length, packed, heads, dk, dv):
    """At most one fp32 state for every 128 tokens of a head, and two more a sequence."""
    from visionhope_b200 import _lib

    lib = _lib.load()
    a, p, keep = _args(batch=batch, length=length, heads=heads, key_dim=dk, value_dim=dv, seq_offsets=(lambda p: p) if packed else None)
    tokens = length * (1 if packed else batch)
    most = (tokens // 128 + 2 * batch) * heads * dk * dv * 4
    for f in (lib.vh_linear_attention_fwd_workspace_bytes, lib.vh_linear_attention_bwd_workspace_bytes):
        assert 0 <= f(ctypes.byref(a)) <= most and _err() == ""
