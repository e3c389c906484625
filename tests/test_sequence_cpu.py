"""Refusals of the sequence operators' C entry points (no device is touched) and their reference's self-consistency."""
import ctypes as C

import pytest
import torch

import sequence_reference as ref


@pytest.fixture(scope="module")
def lib():
    from sound_event_detection_amd import _lib
    return _lib.lib()


P = C.c_void_p(4096)            # a pointer that a refused call never follows


def norm(lib, x=P, y=C.c_void_p(1 << 40), clips=2, frames=3, inner=1, channels=8, groups=2, eps=1e-5, act=0, dtype=0, ws=P, ws_bytes=1 << 20):
    return lib.sedmi_group_norm(x, None, None, None, y, clips, frames, inner, channels, groups, eps, act, dtype, ws, ws_bytes,
                                None)


def test_group_norm_refusals(lib):
    assert norm(lib, groups=3) == -1 and b"multiple of groups" in lib.sedmi_last_error()
    assert norm(lib, groups=0) == -1 and norm(lib, channels=0) == -1
    assert norm(lib, dtype=3) == -1 and norm(lib, dtype=-1) == -1
    assert norm(lib, act=4) == -1 and b"activation" in lib.sedmi_last_error()
    assert norm(lib, eps=-1.0) == -1 and norm(lib, eps=float("nan")) == -1
    assert norm(lib, clips=-1) == -1 and norm(lib, frames=-1) == -1 and norm(lib, inner=0) == -1
    assert norm(lib, frames=1 << 40, inner=1 << 20) == -1
    assert norm(lib, x=None) == -1 and b"null" in lib.sedmi_last_error()
    assert norm(lib, clips=4, frames=5000, channels=1024, groups=32, ws=None) == -3
    assert norm(lib, clips=4, frames=5000, channels=1024, groups=32, ws_bytes=64) == -3 and b"workspace" in lib.sedmi_last_error()
    assert norm(lib, clips=0) == 0 and norm(lib, frames=0) == 0
    assert lib.sedmi_group_norm_workspace_bytes(2, 3, 1, 8, 3, 0) == 0


def conv(lib, x=P, weight=P, state_in=None, state_out=None, y=P, clips=2, frames=3, channels=8, width=4, act=0, dtype=0):
    return lib.sedmi_causal_conv1d(x, 24, 8, weight, None, None, state_in, state_out, y, clips, frames, channels, width, act,
                                   0, dtype, None)


def test_causal_conv_refusals(lib):
    assert conv(lib, width=0) == -1 and conv(lib, width=9) == -1 and b"width" in lib.sedmi_last_error()
    assert conv(lib, dtype=7) == -1 and conv(lib, act=-1) == -1
    assert conv(lib, clips=-1) == -1 and conv(lib, frames=-2) == -1 and conv(lib, channels=0) == -1
    assert conv(lib, x=None) == -1 and conv(lib, weight=None) == -1 and conv(lib, y=None) == -1
    assert conv(lib, state_in=C.c_void_p(4096), state_out=C.c_void_p(4096 + 32)) == -1
    assert b"overlap" in lib.sedmi_last_error()
    assert conv(lib, clips=0) == 0


def scan_struct(**kw):
    from sound_event_detection_amd import _lib
    a = _lib.ScanArgs()
    a.x = a.dt = a.B = a.C = a.A = a.y = 4096
    a.n_clips, a.frames, a.channels, a.groups, a.states, a.dtype = 2, 3, 8, 2, 16, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


def test_scan_refusals(lib):
    def run(**kw):
        return lib.sedmi_selective_scan(scan_struct(**kw), None, 0, None)
    assert lib.sedmi_selective_scan(None, None, 0, None) == -1
    assert run(states=0) == -1 and run(states=129) == -1 and b"states" in lib.sedmi_last_error()
    assert run(groups=3) == -1 and run(groups=0) == -1 and run(channels=-8) == -1
    assert run(dtype=5) == -1 and run(frames=-1) == -1 and run(n_clips=-1) == -1
    for k in ("x", "dt", "B", "C", "A", "y"):
        assert run(**{k: None}) == -1, k
    assert run(state_in=8192, state_out=8192) == -1 and b"overlap" in lib.sedmi_last_error()
    assert run(state_in=8192, state_out=8192 + 64) == -1
    need = lib.sedmi_selective_scan_workspace_bytes(1, 6000, 64, 1, 16)
    assert need > 0 and run(n_clips=1, frames=6000, channels=64, groups=1) == -3 and b"workspace" in lib.sedmi_last_error()
    assert run(n_clips=0) == 0
    assert lib.sedmi_selective_scan_workspace_bytes(2, 3, 8, 3, 16) == 0


def test_step_refusals(lib):
    def run(**kw):
        return lib.sedmi_selective_step(scan_struct(**{"frames": 1, "state_in": 8192, "state_out": 8192, **kw}), None)
    assert run(frames=2) == -1 and run(frames=0) == -1
    assert run(state_out=16384) == -1 and run(state_in=None) == -1
    assert run(state_in=None, state_out=None) == -1
    assert run(lengths=4096) == -1 and run(reverse=1) == -1
    assert run(x=None) == -1 and run(states=200) == -1
    assert run(n_clips=0) == 0


def test_scan_arguments_have_the_layout_of_the_header():
    from sound_event_detection_amd import _lib
    assert C.sizeof(_lib.ScanArgs) == 12 * 8 + 3 * 16 + 2 * 24 + 2 * 8 + 6 * 4
    assert _lib.ScanArgs.n_clips.offset == 12 * 8 + 3 * 16 + 2 * 24
    a = _lib.ScanArgs(*range(1, 13), (13, 14), (15, 16), (17, 18), (19, 20, 21), (22, 23, 24), 25, 26, 27, 28, 29, 30, 1, 0)
    assert bytes(a) == _lib.pack_scan_args(*range(1, 31), True, False)


def test_cpu_tensors_are_refused():
    from sound_event_detection_amd import _lib, sequence
    x = torch.zeros(2, 3, 8)
    with pytest.raises(_lib.SedmiError):
        sequence.group_norm(x, 2)
    with pytest.raises(_lib.SedmiError):
        sequence.causal_conv1d(x, torch.zeros(8, 4))
    with pytest.raises(_lib.SedmiError):
        sequence.selective_step(x[:, 0], x[:, 0], torch.zeros(8, 4), torch.zeros(2, 4), torch.zeros(2, 4), torch.zeros(2, 8, 4))


def test_reference_reverse_is_the_flipped_clip():
    g = torch.Generator().manual_seed(1)
    x, dt = torch.randn(1, 9, 3, generator=g), torch.rand(1, 9, 3, generator=g)
    A, B, D = -torch.rand(3, 2, generator=g), torch.randn(1, 9, 2, generator=g), torch.randn(3, generator=g)
    y, _, h, _ = ref.selective_scan(x, dt, A, B, B, D, reverse=True)
    f, _, k, _ = ref.selective_scan(x.flip(1), dt.flip(1), A, B.flip(1), B.flip(1), D)
    assert torch.allclose(y.flip(1), f) and torch.allclose(h, k)
    w = torch.randn(3, 4, generator=g)
    y, _, s = ref.causal_conv1d(x, w, reverse=True)
    f, _, r = ref.causal_conv1d(x.flip(1), w)
    assert torch.allclose(y.flip(1), f) and torch.equal(s, r)
