"""The sequence operators at the sizes and values where one of their kernels' forms begins or ends."""
import pytest
import torch

import sequence_edges as edges
import sequence_reference as ref
from test_gpu_sequence import BF16, F16, F32, TYPES, gpu, layer, layer_weights, on_gpu, rand, scan_inputs, seq  # noqa: F401  (seq: fixture)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("dtype,c,groups", [(F32, 347823, 115941), (BF16, 594811, 84973), (F16, 594811, 84973)])
def test_group_norm_of_very_many_narrow_groups(seq, dtype, c, groups):
    # more column blocks than a block has groups; groups narrower than a vector
    x, w, b = rand(101, 1, 3, 1, c, dtype=dtype), rand(102, c, offset=1.0), rand(103, c)
    _, depth = edges.two_launch_depth(1, 3, c, groups, dtype)
    y, bound = edges.group_norm(x, groups, w, b, 1e-3, depth)
    ref.check(seq.group_norm(x.cuda(), groups, w.cuda(), b.cuda(), eps=1e-3), y, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", edges.FAR_SHAPES)
def test_group_norm_of_rows_far_from_zero_in_two_launches(seq, shape, dtype):
    # test_sequence_edges_cpu.py: squares about zero are off by more than this bound
    from sound_event_detection_amd import _lib
    n, t, inner, c, groups = shape
    assert _lib.lib().sedmi_group_norm_workspace_bytes(n, t, inner, c, groups, TYPES.index(dtype)) > 0
    x, w, b = edges.far_input(shape)
    x = x.to(dtype)
    chunks, depth = edges.two_launch_depth(n, t * inner, c, groups, dtype)
    assert chunks > 1 or n == 512
    y, bound = edges.group_norm(x, groups, w, b, 1e-5, depth)
    ref.check(seq.group_norm(x.cuda(), groups, w.cuda(), b.cuda()), y, bound)


# groups of 4097 .. 8192 vectors, eight to a thread; the second's rows end inside a vector
SLABS = {F32: [(256, 600, 1, 32, 1), (128, 300, 2, 60, 2)], F16: [(256, 1100, 1, 32, 1), (128, 600, 2, 60, 2)]}
SLABS[BF16] = SLABS[F16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("ragged", [False, True])
def test_group_norm_of_groups_that_fill_a_workgroup(seq, which, ragged, dtype):
    n, t, inner, c, groups = SLABS[dtype][which]
    each, depth = edges.one_launch_depth(t * inner, c, groups, dtype)
    assert 4 < each <= 8
    x = rand(104, n, t, inner, c, dtype=dtype, scale=1.3, offset=0.4)
    x[3] += 60                                                     # far from zero
    w, b = rand(105, c, offset=1.0), rand(106, c)
    lengths = ([0, 1, t - 1, t, t // 2, t // 3, 7, t] * (n // 8)) if ragged else None
    y, bound = edges.group_norm(x, groups, w, b, 1e-4, depth, "silu", lengths)
    got = seq.group_norm(x.cuda(), groups, w.cuda(), b.cuda(), eps=1e-4, activation="silu", lengths=lengths)
    ref.check(got, y, bound)


# --------------------------------------------------------------------------------------------------- causal convolution
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,n,t,c,rows", [(F32, 64, 250, 517, 16), (F32, 64, 250, 1037, 32), (BF16, 128, 251, 531, 16),
                                              (F16, 128, 251, 1051, 32)])
def test_causal_conv_in_long_runs(seq, dtype, n, t, c, rows, reverse):
    vectors, length = -(-c // (4 if dtype == F32 else 8)), 8
    while length < 32 and n * -(-t // length) * vectors > 262144:
        length *= 2
    assert length == rows
    lengths = [0, 1, 2, 15, 16, 17, 33, t - 1] + [t, t // 2, t // 3, 47] * ((n - 8) // 4)
    x, w, b, s = rand(107, n, t, c, dtype=dtype), rand(108, c, 4), rand(109, c), rand(160, n, 3, c, dtype=dtype)
    y, bound, last = ref.causal_conv1d(x, w, b, "silu", s, lengths, reverse)
    for i, v in enumerate(lengths):
        x[i, v:] = float("nan")
    got, end = seq.causal_conv1d(*gpu(x, w, b), "silu", s.cuda(), lengths, reverse, return_state=True)
    ref.check(got, y, bound)
    assert torch.equal(end.cpu(), last)


# ------------------------------------------------------------------------------- more work items than one launch can have
def repeats(y, base):
    """Whether the rows of y are those of base again and again, compared a part at a time."""
    n = base.shape[0]
    return all(bool((part.view(-1, *base.shape) == base).all()) for part in y.split(n << 10))


def test_group_norm_of_more_groups_than_a_launch_holds(seq):
    n, c, groups = 1 << 18, 1024, 64                               # 2^24 workgroups of 256 threads
    base, w, b = rand(110, 64, c, dtype=F16), rand(111, c, offset=1.0), rand(112, c)
    y, bound = ref.group_norm(base, groups, w, b, activation="silu")
    got = seq.group_norm(base.cuda().repeat(n // 64, 1), groups, w.cuda(), b.cuda(), activation="silu")
    ref.check(got[:64], y, bound)
    assert repeats(got, got[:64])
    lengths = torch.ones(n, dtype=torch.int64, device="cuda")
    lengths[-3:] = 0
    got = seq.group_norm(base.cuda().repeat(n // 64, 1)[:, None], groups, w.cuda(), b.cuda(), activation="silu", lengths=lengths)
    ref.check(got[:64, 0], y, bound)
    ref.check(got[-64:-3, 0], y[:-3], bound[:-3])
    assert not bool(got[-3:].any())


def test_causal_conv_of_more_clips_than_a_launch_holds(seq):
    n, c, k = 1 << 22, 6152, 2                                     # 4 workgroups a clip; one row of x for all
    x, w = rand(113, 1, 1, c, dtype=F16), rand(115, c, k)
    got = seq.causal_conv1d(x.cuda().expand(n, 1, c), w.cuda())
    y, bound, _ = ref.causal_conv1d(x, w)
    ref.check(got[:1], y, bound)
    assert all(bool((part == got[0]).all()) for part in got.split(1 << 18))


def test_scan_of_more_clips_than_a_launch_holds(seq):
    n, c, m = 1 << 22, 4, 17                                       # 4 groups of one channel: 4 workgroups a clip
    d = scan_inputs(116, 16, 1, c, m, 4, F16)
    y, bound, _, _ = ref.selective_scan(**d, dt_softplus=True)
    big = {k: v if k in ("A", "D", "dt_bias") else v.repeat(n // 16, *[1] * (v.dim() - 1)) for k, v in on_gpu(d).items()}
    got = seq.selective_scan(**big, dt_softplus=True)
    ref.check(got[:16], y, bound)
    assert repeats(got, got[:16])


def test_step_of_more_streams_than_a_launch_holds(seq):
    n, c, m = 1 << 22, 4, 33
    d, state = scan_inputs(117, 16, None, c, m, 4, F16), rand(118, 16, c, m)
    one = {k: v if k in ("A", "D", "dt_bias") else v[:, None] for k, v in d.items()}
    y, bound, end, end_bound = ref.selective_scan(**one, dt_softplus=True, state=state)
    big = {k: v if k in ("A", "D", "dt_bias") else v.repeat(n // 16, *[1] * (v.dim() - 1)) for k, v in on_gpu(d).items()}
    held = state.cuda().repeat(n // 16, 1, 1)
    got = seq.selective_step(**big, state=held, dt_softplus=True)
    ref.check(got[:16], y[:, 0], bound[:, 0])
    ref.check(held[:16], end, end_bound, "state")
    assert repeats(got, got[:16]) and repeats(held, held[:16])


# ------------------------------------------------------------------------------------------------- infinities in the scan
def positive_scan(seed, n, t, c, m, dtype):
    """Inputs whose sums over states have terms of one sign, so that an infinite input gives an infinite output."""
    d = scan_inputs(seed, n, t, c, m, 1, dtype)
    return {k: v if k in ("A", "dt", "dt_bias") else v.abs() for k, v in d.items()}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", ["x", "dt"])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 12, 16, 17, 33, 100])
def test_scan_infinite_input_gives_infinite_output(seq, m, what, dtype):
    # state counts between those that the lanes hold: what stands in the places left over must not reach the output
    d = positive_scan(120, 2, 40, 19, m, dtype)
    d[what][1, 7, 3] = float("inf")
    for skip in (d["D"], None):
        d["D"] = skip
        y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True)
        if skip is None:
            y[1, 7, 3] = float("inf")                              # the oracle's 0 * inf of the missing D
        assert bool(torch.isinf(y[1, 7:, 3]).all()) and bool(torch.isinf(end[1, 3]).all())
        got, last = seq.selective_scan(**on_gpu(d), dt_softplus=True, return_state=True)
        ref.check(got, y, bound)
        ref.check(last, end, end_bound, "state")
        state = torch.zeros(2, 19, m, device="cuda")
        one = {k: v if v is None or k in ("A", "D", "dt_bias") else v[:, 7].contiguous() for k, v in d.items()}
        got = seq.selective_step(**on_gpu(one), state=state, dt_softplus=True)
        assert float(got[1, 3]) == float("inf") and bool(torch.isinf(state[1, 3]).all())
        assert int(torch.isfinite(got).sum()) == got.numel() - 1


# ---------------------------------------------------------------------------------------------- runs of a long time axis
def is_split(n, t, c, groups, m):
    from sound_event_detection_amd import _lib
    return _lib.lib().sedmi_selective_scan_workspace_bytes(n, t, c, groups, m) > 0


def test_joined_runs_of_growing_states(seq):
    # rates above zero: a run's growth 2^184 has no float32, what it multiplies has
    n, t, c, m = 1, 300, 24, 4
    assert is_split(n, t, c, 1, m)
    d = positive_scan(130, n, t, c, m, F32)
    d["dt"], d["dt_bias"], d["z"] = torch.ones(n, t, c), None, None
    d["A"] = torch.full((c, m), 2.0)
    d["x"][:, :290] = 0.0                                          # no state until the last frames
    y, bound, end, end_bound = ref.selective_scan(**d)
    got, last = seq.selective_scan(**on_gpu(d), return_state=True)
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")
    state = torch.full((n, c, m), 2.0 ** -120)                     # ends at 2^110 after 80 frames
    y, bound, end, end_bound = ref.selective_scan(**d, state=state, lengths=[80])
    got, last = seq.selective_scan(**on_gpu(d), state=state.cuda(), lengths=[80], return_state=True)
    assert bool(torch.isfinite(end).all()) and float(end.max()) > 2.0 ** 100
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")


def test_joined_runs_of_an_infinite_state(seq):
    # an infinite state stays infinite, also where a run's decay is below every float32
    n, t, c, m = 2, 300, 24, 4
    assert is_split(n, t, c, 1, m)
    d = positive_scan(131, n, t, c, m, F32)
    d["A"] = torch.full((c, m), -8.0)
    d["x"][1, 5, 3] = float("inf")
    y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True)
    assert bool(torch.isinf(y[1, 5:, 3]).all())
    got, last = seq.selective_scan(**on_gpu(d), dt_softplus=True, return_state=True)
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m", [1, 2, 4, 5, 17, 32, 33, 64, 100, 128])
def test_joined_runs_of_all_state_counts(seq, m, dtype, reverse):
    n, t, c, lengths = 2, 300, 24, [300, 170]
    assert is_split(n, t, c, 2, m)
    d = scan_inputs(132, n, t, c, m, 2, dtype)
    d["A"][:4] *= 1e-3                                             # channels that remember across the runs
    state = rand(133, n, c, m)
    y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True, state=state, lengths=lengths, reverse=reverse)
    got, last = seq.selective_scan(**on_gpu(d), dt_softplus=True, state=state.cuda(), lengths=lengths, reverse=reverse,
                                   return_state=True)
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")


@pytest.mark.parametrize("what", ["x", "dt", "state"])
def test_joined_runs_keep_nan_in_its_channel(seq, what):
    n, t, c, m = 2, 300, 24, 5
    d, state = scan_inputs(134, n, t, c, m, 1, F32), rand(135, n, c, m)
    if what == "state":
        state[1, 3, 2] = float("nan")
    else:
        d[what][1, 100, 3] = float("nan")
    y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True, state=state)
    got, last = seq.selective_scan(**on_gpu(d), dt_softplus=True, state=state.cuda(), return_state=True)
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")


# ------------------------------------------------------------------------------------------------------------ from audio
def test_events_from_audio_through_a_layer_of_them(seq):
    # recordings of unequal length: mel features, a layer in both directions, frame probabilities, events
    import numpy as np
    from oracle import decode as odec
    from sound_event_detection_amd import evaluation, feature_extraction, synth
    audio = torch.from_numpy(synth.synth_clips(0, 3)).cuda()
    x = feature_extraction.mel_features(audio, 16000, 2048, 128, 320, 640, log=True)
    n, t, c = x.shape
    lengths, classes = [t, 300, 77], 5
    w, head = layer_weights(c, 16, 4), rand(170, 2 * c, classes, scale=c ** -0.5)
    on_device = torch.tensor(lengths, device="cuda")
    both = torch.cat([layer(seq, w, x, on_device, reverse)[0] for reverse in (False, True)], -1)
    probs = torch.sigmoid(both @ head.cuda())

    w64 = {k: v.cpu().double() for k, v in w.items()}
    u = ref.group_norm(x.cpu(), 4, w64["norm_w"], w64["norm_b"], activation="silu", lengths=lengths)[0]
    sides = []
    for reverse in (False, True):
        v = ref.causal_conv1d(u, w64["conv_w"], w64["conv_b"], "silu", lengths=lengths, reverse=reverse)[0]
        bc = v @ w64["to_bc"]
        sides.append(ref.selective_scan(v, v @ w64["to_dt"], w64["A"], bc[..., :16], bc[..., 16:], w64["D"], u, w64["dt_bias"],
                                        True, lengths=lengths, reverse=reverse)[0])
    want = torch.sigmoid(torch.cat(sides, -1) @ head.double())
    assert float((probs.cpu().double() - want).abs().max()) < 1e-3         # the models' own bound on frame probabilities

    seg, cls, on, off = evaluation.decode_recordings(probs.view(-1, classes), [t] * n, lengths)
    events = [(i, *e) for i in range(n) for e in odec.decode_events(odec.threshold(probs[i].cpu().numpy()), lengths[i])]
    assert len(events) > 10 and events == list(zip(*(np.asarray(v).tolist() for v in (seg, cls, on, off))))


# ------------------------------------------------------------------------------------------------------ forward derivatives
def test_calls_refuse_tensors_with_a_tangent(seq):
    from torch.autograd import forward_ad
    x, w = torch.ones(2, 5, 8, device="cuda"), torch.ones(8, 4, device="cuda")
    d = on_gpu(scan_inputs(140, 2, 5, 8, 4, 1, F32))
    one = {k: v if k in ("A", "D", "dt_bias") else v[:, 0] for k, v in d.items()}
    conv_state, scan_state = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: seq.group_norm(dual(x), 2), lambda: seq.group_norm(x, 2, bias=dual(w[:, 0])),
                     lambda: seq.causal_conv1d(x, dual(w)), lambda: seq.causal_conv1d_step(x[:, 0], dual(conv_state), w),
                     lambda: seq.selective_scan(**{**d, "dt": dual(d["dt"])}),
                     lambda: seq.selective_scan(**{**d, "A": dual(d["A"])}),
                     lambda: seq.selective_step(**one, state=dual(scan_state))):
            with pytest.raises(RuntimeError, match="inference-only"):
                call()
        assert seq.group_norm(x, 2).shape == x.shape               # others are served
    assert not bool(conv_state.any()) and not bool(scan_state.any())


# ------------------------------------------------------------------------------------------------------- states in place
def test_steps_count_as_changes_of_their_state(seq):
    x, w = rand(150, 2, 8).cuda(), rand(151, 8, 4).cuda()
    d = on_gpu(scan_inputs(152, 2, None, 8, 4, 1, F32))
    for state, call in ((torch.zeros(2, 3, 8, device="cuda"), lambda s: seq.causal_conv1d_step(x, s, w)),
                        (torch.zeros(2, 8, 4, device="cuda"), lambda s: seq.selective_step(**d, state=s, dt_softplus=True))):
        factor = torch.ones_like(state, requires_grad=True)
        out = (factor * state).sum()                               # keeps the state for its backward pass
        call(state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()
        before = state._version
        call(state[:1].expand(2, -1, -1).contiguous())             # another tensor
        assert state._version == before
        with torch.inference_mode():
            call(state.clone())                                    # has no versions
            call(state)
        assert state._version == before + 1


# ------------------------------------------------------------------------------------------------------------- refusals
def test_group_norm_refuses_a_fraction_of_a_group(seq):
    x = torch.zeros(2, 5, 8, device="cuda")
    for groups in (2.7, 8.5, "2"):
        with pytest.raises(ValueError, match="do not divide"):
            seq.group_norm(x, groups)
    for groups in (2.0, torch.tensor(2)):
        assert seq.group_norm(x, groups).shape == x.shape
