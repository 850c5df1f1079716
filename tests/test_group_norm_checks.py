"""What the group norm entry points answer without a GPU: the argument struct's layout, sizes and refusals."""
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
    a = _lib.VhGroupNormArgs(x=p, x_sample_stride=64 * 64, x_pixel_stride=64, y=p, samples=2, pixels=64, eps=1e-5, dtype=1,
                             channels=64, groups=8, activation=1)
    for n, v in kw.items():
        setattr(a, n, v(p) if callable(v) else v)
    return a, p, keep


def _err():
    from visionhope_b200 import _lib

    return _lib.load().vh_last_error().decode()


def test_struct_layout(tmp_path):
    from visionhope_b200 import _lib
    from visionhope_b200.utils import group_norm  # noqa: F401

    names = [n for n, _ in _lib.VhGroupNormArgs._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "vhope.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu\\n", offsetof(vh_group_norm_args, {n}));\n' for n in names)
                   + 'printf("%zu\\n", sizeof(vh_group_norm_args));\nreturn 0; }\n')
    exe = tmp_path / "o"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    want = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert want[:-1] == [getattr(_lib.VhGroupNormArgs, n).offset for n in names]
    assert want[-1] == ctypes.sizeof(_lib.VhGroupNormArgs) == group_norm._ARGS.size


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null"), (dict(dtype=5), "dtype"), (dict(samples=0), "positive"), (dict(pixels=0), "positive"),
    (dict(channels=0), "positive"), (dict(groups=0), "positive"), (dict(groups=7), "multiple of groups"), (dict(activation=3), "activation"),
    (dict(channels=1 << 21, groups=1), "2^20"), (dict(pixels=1 << 31), "2^31"), (dict(x=lambda p: p + 1), "misaligned"),
    (dict(weight=lambda p: p + 2), "misaligned"), (dict(mean=lambda p: p), "together")])
def test_refused_arguments(change, text):
    from visionhope_b200 import _lib

    lib = _lib.load()
    a, p, keep = _args(**change)
    assert lib.vh_group_norm_fwd(ctypes.byref(a), p, 1 << 40, None) < 0 and text in _err()
    assert lib.vh_group_norm_bwd(ctypes.byref(a), p, p, None, p, p, p, 1 << 40, None) < 0 and text in _err()


def test_refused_workspaces_and_gradients():
    from visionhope_b200 import _lib

    lib = _lib.load()
    a, p, keep = _args(mean=lambda p: p, rstd=lambda p: p)
    need = lib.vh_group_norm_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.vh_group_norm_bwd(ctypes.byref(a), p, p, None, p, p, p, need // 2 - 1, None) < 0 and "workspace" in _err()
    assert lib.vh_group_norm_bwd(ctypes.byref(a), p, p, p, p, p, p, need, None) < 0 and "null" in _err()
    assert lib.vh_group_norm_bwd(ctypes.byref(a), None, p, None, p, p, p, need, None) < 0 and "null" in _err()
    assert lib.vh_group_norm_bwd(ctypes.byref(a), p, p + 1, None, p, p, p, need, None) == -5
    assert lib.vh_group_norm_bwd(ctypes.byref(a), p, p, None, p + 2, p, p, need, None) == -5
    a, p, keep = _args()
    assert lib.vh_group_norm_bwd(ctypes.byref(a), p, p, None, p, p, p, need, None) < 0 and "null" in _err()
    a, p, keep = _args(y=None)
    assert lib.vh_group_norm_fwd(ctypes.byref(a), p, 1 << 40, None) < 0 and "null" in _err()
    assert lib.vh_group_norm_fwd_workspace_bytes(None) == 0 and lib.vh_group_norm_fwd(None, None, 0, None) < 0


@pytest.mark.parametrize("channels,groups", [(64, 8), (91, 7), (2048, 16), (4096, 1), (96, 96)])
@pytest.mark.parametrize("samples,pixels", [(1, 1), (50176, 1), (64, 3136), (2, 65536), (1, 1 << 30), (100000, 49)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspaces(channels, groups, samples, pixels, dtype):
    """Some numbers a channel for each sample or block, never as much as the data."""
    from visionhope_b200 import _lib

    lib = _lib.load()
    a, p, keep = _args(channels=channels, groups=groups, samples=samples, pixels=pixels, dtype=dtype)
    f, b = lib.vh_group_norm_fwd_workspace_bytes(ctypes.byref(a)), lib.vh_group_norm_bwd_workspace_bytes(ctypes.byref(a))
    assert _err() == "" and 0 <= f <= 8 * channels * (4096 + 3 * samples) and 0 < b <= 8 * channels * (4096 + 4 * samples)
