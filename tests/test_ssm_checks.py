"""What the selective state space entry points answer without a GPU: sizes and refusals at the edges
of their arguments' ranges."""
import ctypes

import pytest

from tests.test_oracle_ssm import _conv_args, _err, _fake, _scan_args


def _bwd(lib, p, fwd):
    return lib.VhSsmScanBwdArgs(fwd=fwd, grad_y=p, grad_final=None, grad_u=p, grad_delta=p, grad_z=p, grad_b=p, grad_c=p,
                                grad_a=p, grad_d_skip=p, grad_delta_bias=p, grad_initial=None)


@pytest.mark.parametrize("states", [4, 16, 64])
@pytest.mark.parametrize("batch", [1, 2, 5000])
@pytest.mark.parametrize("packed", [False, True])
def test_sizes_for_sequences_without_tokens(packed, batch, states):
    """A length of 0 is allowed: sizes come back, and the host is still there."""
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    a = _scan_args(_lib, p, length=0, batch=batch, states=states, seq_offsets=p if packed else None, checkpoints=p)
    assert lib.vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a)) >= 0 and _err(lib) == ""
    assert lib.vh_ssm_scan_checkpoint_bytes(ctypes.byref(a)) >= 0
    assert lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(_bwd(_lib, p, a))) > 0 and _err(lib) == ""
    c = _conv_args(_lib, p, length=0, batch=batch, seq_offsets=p if packed else None)
    assert lib.vh_short_conv_bwd_workspace_bytes(ctypes.byref(c)) > 0


@pytest.mark.parametrize("change", [dict(states=12), dict(states=3), dict(states=516), dict(states=1 << 20), dict(states=-16),
                                    dict(dtype=9), dict(batch=0), dict(groups=3), dict(length=-1), dict(length=1 << 31)])
def test_sizes_of_unsupported_scans_are_zero(change):
    """A query with arguments that the operator refuses gives 0, whatever the values."""
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    a = _scan_args(_lib, p, checkpoints=p, **change)
    assert lib.vh_ssm_scan_checkpoint_bytes(ctypes.byref(a)) == 0
    assert lib.vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(_bwd(_lib, p, a))) == 0
    assert lib.vh_ssm_scan_checkpoint_bytes(None) == 0


def test_offsets_and_slots_do_not_wrap():
    """int64 offsets and slots past int32 stay outside the tokens and the cache."""
    import torch

    from visionhope_b200.ssm_core import _args

    cpu = torch.device("cpu")
    far = torch.tensor([-(1 << 32), -1, 0, 7, (1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 62])
    want = torch.tensor([-1, -1, 0, 7] + [(1 << 31) - 1] * 4, dtype=torch.int32)
    assert torch.equal(_args.offsets_like(far, cpu), want)
    assert torch.equal(_args.slot_index(far, 8, cpu), want)
    near = torch.arange(10, dtype=torch.int32)[::2]
    assert torch.equal(_args.offsets_like(near, cpu), near) and _args.offsets_like(near, cpu).is_contiguous()
    whole = near.contiguous()
    assert _args.offsets_like(whole, cpu) is whole


def test_parameters_and_states_need_four_bytes():
    """fp32 arrays of the sequence entry points may lie anywhere in a larger buffer; what is moved
    sixteen bytes at a time (checkpoints, workspaces, the step's rates and states) may not."""
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    names = ("a", "d_skip", "delta_bias", "initial_state", "final_state")

    def scan(**kw):
        return _scan_args(_lib, p, checkpoints=kw.pop("checkpoints", p), **kw)

    def query(a):
        lib.vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a))
        return _err(lib)

    assert query(scan(**{n: p + 4 for n in names})) == ""
    for n in names:
        assert "misaligned" in query(scan(**{n: p + 2}))
    assert "checkpoints" in query(scan(checkpoints=p + 4))
    a = _bwd(_lib, p, scan(**{n: p + 4 for n in names}))
    a.grad_final = a.grad_initial = a.grad_a = a.grad_d_skip = a.grad_delta_bias = p + 4
    assert lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(a)) > 0 and _err(lib) == ""
    a.grad_final = p + 2
    assert lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(a)) == 0 and "misaligned" in _err(lib)
    assert lib.vh_ssm_scan_step(ctypes.byref(scan(a=p + 4)), p, p, None, 4, None) == -5
    assert lib.vh_ssm_scan_step(ctypes.byref(scan()), p + 4, p, None, 4, None) == -5


@pytest.mark.parametrize("states", [4, 8, 16, 32, 64])
@pytest.mark.parametrize("batch,length,channels,packed", [(64, 3136, 1024, False), (2, 16384, 384, False), (8, 196, 512, False),
                                                          (1000, 20000, 512, True), (17, 8192, 1024, True)])
def test_memory_is_as_documented(batch, length, channels, packed, states):
    """Checkpoints and workspaces per element, plus what segments and packed sequences add."""
    from visionhope_b200 import _lib

    lib, (p, keep) = _lib.load(), _fake()
    a = _scan_args(_lib, p, batch=batch, length=length, channels=channels, states=states, seq_offsets=p if packed else None,
                   checkpoints=p)
    elements = channels * length * (1 if packed else batch)
    per = batch * -(-channels * states // 512) if packed else 0  # sequences by tiles
    fwd, ck = lib.vh_ssm_scan_fwd_workspace_bytes(ctypes.byref(a)), lib.vh_ssm_scan_checkpoint_bytes(ctypes.byref(a))
    bwd = lib.vh_ssm_scan_bwd_workspace_bytes(ctypes.byref(_bwd(_lib, p, a)))
    assert 0 <= fwd <= (20 << 20) + 3072 * per
    assert elements * states // 8 <= ck + 2048 * per <= elements * states // 8 * 1.2 + 4096 * per
    assert 0 <= bwd - elements * states ** 2 // 64 <= (40 << 20) + 6144 * per
