"""Parts of the sequence operators that no device is needed for."""
import test_sequence_cpu as cpu
from test_sequence_cpu import lib  # noqa: F401  (fixture)


def test_a_clip_that_no_launch_can_hold_is_refused(lib):
    def scan(entry, *ws, **kw):
        return entry(cpu.scan_struct(channels=1 << 24, groups=1 << 24, frames=1, n_clips=1, **kw), *ws, None)
    assert scan(lib.sedmi_selective_scan, None, 0, states=17) == -1 and b"workgroups" in lib.sedmi_last_error()
    assert scan(lib.sedmi_selective_step, states=4, state_in=8192, state_out=8192) == -1
    assert b"workgroups" in lib.sedmi_last_error()
    assert cpu.conv(lib, clips=1, frames=1 << 38, channels=1) == -1 and b"workgroups" in lib.sedmi_last_error()
