"""Parts of the sequence operators that no device is needed for."""
import pytest
import torch
from torch.autograd import forward_ad

import test_sequence_cpu as cpu
from test_sequence_cpu import lib  # noqa: F401  (fixture)


def test_a_clip_that_no_launch_can_hold_is_refused(lib):
    def scan(entry, *ws, **kw):
        return entry(cpu.scan_struct(channels=1 << 24, groups=1 << 24, frames=1, n_clips=1, **kw), *ws, None)
    assert scan(lib.sedmi_selective_scan, None, 0, states=17) == -1 and b"workgroups" in lib.sedmi_last_error()
    assert scan(lib.sedmi_selective_step, states=4, state_in=8192, state_out=8192) == -1
    assert b"workgroups" in lib.sedmi_last_error()
    assert cpu.conv(lib, clips=1, frames=1 << 38, channels=1) == -1 and b"workgroups" in lib.sedmi_last_error()


def test_tensors_with_a_tangent_are_refused():
    from sound_event_detection_amd import sequence
    x = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        sequence._refuse_grad("the call", x, None)
        with pytest.raises(RuntimeError, match="the call is inference-only"):
            sequence._refuse_grad("the call", x, None, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="the call is inference-only"):
            sequence._refuse_grad("the call", dual)                # no_grad leaves forward mode on
        with torch.inference_mode():
            sequence._refuse_grad("the call", dual)                # which switches it off
    sequence._refuse_grad("the call", x)


def test_the_package_names_the_module():
    import sound_event_detection_amd
    assert "sequence" in sound_event_detection_amd.__all__
