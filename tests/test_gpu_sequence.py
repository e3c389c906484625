"""The sequence operators (group norm, short causal convolution, selective state space scan) against their definitions
in float64, with error bounds derived in tests/sequence_reference.py."""
import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


@pytest.fixture(scope="module")
def seq():
    from sound_event_detection_amd import sequence
    return sequence


def rand(seed, *shape, dtype=F32, scale=1.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + offset).to(dtype)


def gpu(*ts):
    return [t.cuda() for t in ts]


# ----------------------------------------------------------------------------------------------------------- group norm
NORM_SHAPES = [
    # clips, frames, inner, channels, groups
    (1, 1, 1, 1, 1), (2, 3, 1, 6, 3), (3, 7, 5, 24, 2), (2, 33, 1, 64, 64), (1, 251, 1, 387, 1), (2, 129, 2, 96, 32),
    (5, 40, 3, 40, 5), (2, 9, 1, 2500, 1), (1, 12, 1, 4100, 2), (2, 700, 4, 16, 4), (1, 2100, 1, 256, 8), (3, 50, 1, 7, 7),
    # groups of more than a workgroup's registers: rows in chunks, one group wider than a workgroup, several column
    # blocks, groups that end inside a 16-byte vector, rows of fewer channels than a vector
    (2, 300, 1, 1024, 2), (1, 40, 1, 2500, 1), (1, 60, 1, 4100, 1), (1, 70, 1, 5000, 200), (2, 1100, 1, 60, 10),
    (3, 500, 1, 37, 37), (2, 9000, 1, 5, 1), (1, 700, 1, 3, 3), (1, 9, 1, 2056, 257), (2, 901, 2, 100, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_group_norm(seq, shape, dtype):
    n, t, inner, c, g = shape
    x = rand(1, n, t, inner, c, dtype=dtype, scale=1.3, offset=0.4)
    w, b = rand(2, c, offset=1.0), rand(3, c)
    for act in (None, "silu"):
        got = seq.group_norm(x.cuda(), g, *gpu(w, b), eps=1e-4, activation=act)
        assert got.dtype == dtype
        y, bound = ref.group_norm(x, g, w, b, 1e-4, act)
        ref.check(got, y, bound, f"{shape} {act}")


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
def test_group_norm_activations_and_missing_parameters(seq, act):
    x = rand(4, 3, 20, 48, scale=2.0)
    y, bound = ref.group_norm(x, 6, activation=act)
    ref.check(seq.group_norm(x.cuda(), 6, activation=act), y, bound)
    flat = rand(5, 9, 32)
    y, bound = ref.group_norm(flat, 4, activation=act)
    ref.check(seq.group_norm(flat.cuda(), 4, activation=act), y, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(6, 37, 1, 64, 8), (6, 37, 3, 20, 1), (6, 600, 8, 32, 4), (6, 300, 1, 1500, 3)])
def test_group_norm_lengths_hide_what_lies_behind_them(seq, shape, dtype):
    n, t, inner, c, g = shape
    lengths = [0, 1, t, t - 1, t // 2, t + 50]                     # the last is taken as t
    x = rand(6, n, t, inner, c, dtype=dtype)
    hidden = x.clone()
    for i, k in enumerate(lengths):
        hidden[i, k:] = float("nan")
        hidden[i, k:, :, ::3] = float("inf")
    w, b = rand(7, c), rand(8, c)
    y, bound = ref.group_norm(x, g, w, b, activation="relu", lengths=lengths)
    got = seq.group_norm(hidden.cuda(), g, *gpu(w, b), activation="relu", lengths=torch.tensor(lengths, dtype=torch.int32))
    ref.check(got, y, bound)
    assert not bool(seq.group_norm(x.cuda(), g, lengths=[-3] * n).any())


def test_group_norm_far_from_zero_and_constant(seq):
    # the mean is 500 standard deviations away: squares summed about zero would lose all digits of the variance
    x = rand(9, 2, 400, 32, scale=0.25, offset=125.0)
    x[1] += 0.0
    x[1, 0] = 0.0                                                  # an outlying first row
    y, bound = ref.group_norm(x, 4)
    ref.check(seq.group_norm(x.cuda(), 4), y, bound)
    const = torch.full((2, 50, 16), 3.0)
    assert not bool(seq.group_norm(const.cuda(), 2).any())
    x = rand(10, 2, 30, 16)
    x[1, 3, 5] = float("inf")
    got = seq.group_norm(x.cuda(), 2).cpu()
    assert bool(torch.isnan(got[1, :, :8]).all()) and bool(torch.isfinite(got[1, :, 8:]).all())
    assert bool(torch.isfinite(got[0]).all())


def test_group_norm_other_layouts_and_empty(seq):
    x = rand(11, 3, 24, 10, 6).permute(0, 2, 3, 1)                 # channels first in memory
    y, bound = ref.group_norm(x, 4)
    ref.check(seq.group_norm(x.cuda(), 4), y, bound)
    wide = rand(12, 4, 11, 90, dtype=F16).cuda()
    y, bound = ref.group_norm(wide[:, :, 7:40].cpu(), 3)
    ref.check(seq.group_norm(wide[:, :, 7:40], 3), y, bound)
    for shape in ((0, 5, 8), (2, 0, 8)):
        assert seq.group_norm(torch.empty(shape, device="cuda"), 2).shape == shape


# --------------------------------------------------------------------------------------------------- causal convolution
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", range(1, 9))
def test_causal_conv_widths(seq, k, dtype):
    n, t, c = 3, 71, 37
    x, w, b, s = rand(20, n, t, c, dtype=dtype), rand(21, c, k), rand(22, c), rand(23, n, k - 1, c, dtype=dtype)
    for state, reverse in ((None, False), (s, False), (s, True)):
        y, bound, last = ref.causal_conv1d(x, w, b, "silu", state, None, reverse)
        got, end = seq.causal_conv1d(*gpu(x, w, b), "silu", None if state is None else state.cuda(), reverse=reverse,
                                     return_state=True)
        ref.check(got, y, bound, f"width {k}")
        assert end.dtype == dtype and torch.equal(end.cpu(), last)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("t", [1, 2, 31, 32, 33, 70])
@pytest.mark.parametrize("c", [1, 8, 130])
def test_causal_conv_lengths(seq, t, c, reverse):
    lengths = [0, 1, 2, 3, t // 2, t, t + 9]
    n, k = len(lengths), 4
    x, w, s = rand(24, n, t, c), rand(25, c, k), rand(26, n, k - 1, c)
    hidden = x.clone()
    for i, v in enumerate(lengths):
        hidden[i, v:] = float("nan")
    y, bound, last = ref.causal_conv1d(x, w, None, None, s, lengths, reverse)
    got, end = seq.causal_conv1d(*gpu(hidden, w), state=s.cuda(), lengths=lengths, reverse=reverse, return_state=True)
    ref.check(got, y, bound)
    assert torch.equal(end.cpu(), last)


def test_causal_conv_slices_in_pieces_and_by_frames(seq):
    n, t, c, k = 4, 90, 50, 4
    wide = rand(27, n, t, 2 * c + 3, dtype=BF16)
    x, w, b = wide[:, :, 3:c + 3], rand(28, c, k), rand(29, c)
    gx, gw, gb = wide.cuda()[:, :, 3:c + 3], w.cuda(), b.cuda()
    y, bound, last = ref.causal_conv1d(x, w, b, "gelu")
    whole, end = seq.causal_conv1d(gx, gw, gb, "gelu", return_state=True)
    ref.check(whole, y, bound)
    parts, state, at = [], None, 0
    for size in (1, 2, 40, 3, 44):
        out, state = seq.causal_conv1d(gx[:, at:at + size], gw, gb, "gelu", state=state, return_state=True)
        parts.append(out)
        at += size
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(state, end)
    state = torch.zeros(n, k - 1, c, dtype=BF16, device="cuda")
    steps = [seq.causal_conv1d_step(gx[:, i], state, gw, gb, "gelu") for i in range(t)]
    assert torch.equal(torch.stack(steps, 1), whole) and torch.equal(state, end)
    turned = gx.transpose(1, 2).contiguous().transpose(1, 2)       # channels not adjacent: copied
    assert torch.equal(seq.causal_conv1d(turned, gw, gb, "gelu"), whole)


def test_causal_conv_without_frames_keeps_the_state(seq):
    s = rand(30, 2, 3, 5).cuda()
    y, end = seq.causal_conv1d(torch.empty(2, 0, 5, device="cuda"), rand(31, 5, 4).cuda(), state=s, return_state=True)
    assert y.shape == (2, 0, 5) and torch.equal(end, s)
    y, end = seq.causal_conv1d(torch.empty(0, 4, 5, device="cuda"), rand(31, 5, 4).cuda(), return_state=True)
    assert y.shape == (0, 4, 5) and end.shape == (0, 3, 5)


# ------------------------------------------------------------------------------------------------------- selective scan
def scan_inputs(seed, n, t, c, m, groups, dtype):
    lead = (n, t) if t is not None else (n,)
    proj = rand(seed, *lead, 3 + 2 * groups * m, dtype=dtype)
    return dict(x=rand(seed + 1, *lead, c, dtype=dtype), dt=rand(seed + 2, *lead, c, dtype=dtype, scale=0.7, offset=-1.5),
                A=-torch.exp(rand(seed + 3, c, m, scale=0.8)), B=proj[..., 3:3 + groups * m].unflatten(-1, (groups, m)),
                C=proj[..., 3 + groups * m:].unflatten(-1, (groups, m)), D=rand(seed + 4, c),
                z=rand(seed + 5, *lead, 2 * c + 1, dtype=dtype)[..., c + 1:], dt_bias=rand(seed + 6, c, scale=0.3))


def on_gpu(d):
    """The same tensors on the GPU with their strides."""
    out = {}
    for k, v in d.items():
        if v is None:
            out[k] = None
        else:
            base = v._base if v._base is not None else v
            while base._base is not None:
                base = base._base
            out[k] = base.cuda().as_strided(v.shape, v.stride(), v.storage_offset())
    return out


def check_scan(seq, d, dtype, what="", **kw):
    y, bound, end, end_bound = ref.selective_scan(**d, **kw)
    state = kw.pop("state", None)
    got, last = seq.selective_scan(**on_gpu(d), **kw, state=None if state is None else state.cuda(), return_state=True)
    assert got.dtype == dtype and last.dtype == F32
    ref.check(got, y, bound, what)
    ref.check(last, end, end_bound, what + " state")
    return got, last


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 3, 4, 5, 8, 12, 16, 17, 32, 40, 64, 128])
def test_scan_state_sizes(seq, m, dtype):
    d = scan_inputs(40, 2, 37, 70, m, 1, dtype)
    check_scan(seq, d, dtype, f"{m} states", dt_softplus=True)


@pytest.mark.parametrize("t", [1, 2, 4, 31, 32, 33, 64, 97])
@pytest.mark.parametrize("c,groups", [(1, 1), (64, 1), (65, 1), (130, 2), (12, 4), (200, 1)])
def test_scan_lengths_of_time_and_channels(seq, t, c, groups):
    d = scan_inputs(41, 2, t, c, 16, groups, F32)
    check_scan(seq, d, F32, dt_softplus=True, state=rand(42, 2, c, 16))


@pytest.mark.parametrize("missing", ["D", "z", "dt_bias", "softplus", "all"])
def test_scan_without_its_optional_parts(seq, missing):
    d = scan_inputs(43, 2, 40, 33, 8, 1, BF16)
    for k in ("D", "z", "dt_bias"):
        if missing in (k, "all"):
            d[k] = None
    if missing in ("softplus", "all"):
        d["dt"] = d["dt"].abs()
    check_scan(seq, d, BF16, dt_softplus=missing not in ("softplus", "all"))
    three = {**d, "B": d["B"].squeeze(2), "C": d["C"].squeeze(2)}
    a = seq.selective_scan(**on_gpu(d), dt_softplus=True)
    assert torch.equal(a, seq.selective_scan(**on_gpu(three), dt_softplus=True))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("t,c", [(5, 20), (70, 20), (700, 70)])
def test_scan_lengths_hide_what_lies_behind_them(seq, t, c, reverse):
    lengths = [0, 1, t // 3, t - 1, t, t + 4]
    n = len(lengths)
    d = scan_inputs(44, n, t, c, 6, 1, F32)
    state = rand(45, n, c, 6)
    y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True, state=state, lengths=lengths, reverse=reverse)
    hidden = {k: v if k in ("A", "D", "dt_bias") else v.clone() for k, v in d.items()}
    for i, v in enumerate(lengths):
        for k in ("x", "dt", "B", "C", "z"):
            hidden[k][i, v:] = float("nan")
            hidden[k][i, v:, ..., ::2] = float("-inf")
    hidden = {k: v.cuda() for k, v in hidden.items()}
    got, last = seq.selective_scan(**hidden, dt_softplus=True, state=state.cuda(), lengths=torch.tensor(lengths).cuda(),
                                   reverse=reverse, return_state=True)
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_a_long_recording_in_runs(seq, dtype, reverse):
    # few channels and a long axis: time is split into runs that are joined
    from sound_event_detection_amd import _lib
    n, t, c, m = 1, 1500, 24, 16
    assert _lib.lib().sedmi_selective_scan_workspace_bytes(n, t, c, 1, m) > 0
    d = scan_inputs(46, n, t, c, m, 1, dtype)
    d["A"][:4] *= 1e-3                                              # channels that remember across the runs
    check_scan(seq, d, dtype, dt_softplus=True, state=rand(47, n, c, m), reverse=reverse)


def test_scan_in_pieces_and_by_frames(seq):
    n, t, c, m = 3, 75, 40, 16
    d = on_gpu(scan_inputs(48, n, t, c, m, 2, F32))
    whole, end = seq.selective_scan(**d, dt_softplus=True, return_state=True)
    parts, state, at = [], None, 0
    for size in (1, 7, 33, 34):
        piece = {k: v if k in ("A", "D", "dt_bias") else v[:, at:at + size] for k, v in d.items()}
        out, state = seq.selective_scan(**piece, dt_softplus=True, state=state, return_state=True)
        parts.append(out)
        at += size
    torch.testing.assert_close(torch.cat(parts, 1), whole, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, end, rtol=1e-5, atol=1e-5)
    state = torch.zeros(n, c, m, device="cuda")
    outs = []
    for i in range(t):
        one = {k: v if k in ("A", "D", "dt_bias") else v[:, i] for k, v in d.items()}
        outs.append(seq.selective_step(**one, state=state, dt_softplus=True))
    torch.testing.assert_close(torch.stack(outs, 1), whole, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, end, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 3, 4, 16, 18, 33, 64, 100, 128])
@pytest.mark.parametrize("n,c,groups", [(1, 5, 1), (3, 130, 2)])
def test_step(seq, n, c, groups, m, dtype):
    d = scan_inputs(49, n, None, c, m, groups, dtype)
    state = rand(50, n, c, m)
    one = {k: v if v is None or k in ("A", "D", "dt_bias") else v[:, None] for k, v in d.items()}
    y, bound, end, end_bound = ref.selective_scan(**one, dt_softplus=True, state=state)
    held = state.cuda()
    got = seq.selective_step(**on_gpu(d), state=held, dt_softplus=True)
    ref.check(got, y[:, 0], bound[:, 0])
    ref.check(held, end, end_bound, "state")
    d["z"] = d["D"] = d["dt_bias"] = None
    d["dt"] = d["dt"].abs()
    one = {k: v if v is None or k == "A" else v[:, None] for k, v in d.items()}
    y, bound, end, end_bound = ref.selective_scan(**one, state=state)
    held = state.cuda()
    ref.check(seq.selective_step(**on_gpu(d), state=held), y[:, 0], bound[:, 0])
    ref.check(held, end, end_bound, "state")


@pytest.mark.parametrize("m", [3, 4, 18, 32])
def test_step_of_many_streams(seq, m):
    # enough streams that a quad of lanes takes four of them; their number is no multiple of four
    n, c = 1027, 6
    d, state = scan_inputs(55, n, None, c, m, 2, F16), rand(56, n, c, m)
    one = {k: v if k in ("A", "D", "dt_bias") else v[:, None] for k, v in d.items()}
    y, bound, end, end_bound = ref.selective_scan(**one, dt_softplus=True, state=state)
    guard = torch.full((n + 8, c, m), 7.0, device="cuda")
    held = guard[4:n + 4]
    held.copy_(state)
    ref.check(seq.selective_step(**on_gpu(d), state=held, dt_softplus=True), y[:, 0], bound[:, 0])
    ref.check(held, end, end_bound, "state")
    assert bool((guard[:4] == 7).all()) and bool((guard[n + 4:] == 7).all())


def test_scan_far_values(seq):
    d = scan_inputs(51, 1, 40, 16, 4, 1, F32)
    d["dt"][0, 5] = 60.0                                           # softplus is the identity, the state is forgotten
    d["dt"][0, 9] = -80.0                                          # a step of e^-80: the state stays
    d["dt"][0, 11] = -200.0
    d["A"][3] = float("-inf")                                      # no memory at all
    d["A"][4] = 0.0                                                # a plain sum
    d["z"][0, 7] = -120.0
    one = on_gpu(d)
    got, last = seq.selective_scan(**one, dt_softplus=True, return_state=True)
    d["A"][3] = -1e30
    y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True)
    bound[..., 3], end_bound[:, 3] = bound[..., 3].nan_to_num(), end_bound[:, 3].nan_to_num()
    keep = [i for i in range(16) if i != 3]
    ref.check(got[..., keep], y[..., keep], bound[..., keep])
    ref.check(last[:, keep], end[:, keep], end_bound[:, keep], "state")
    assert bool(torch.isfinite(got).all())


def test_scan_nan_stays_in_its_channel(seq):
    d = scan_inputs(52, 2, 50, 20, 8, 1, F32)
    d["x"][1, 10, 3] = float("nan")
    y, bound, end, end_bound = ref.selective_scan(**d, dt_softplus=True)
    got, last = seq.selective_scan(**on_gpu(d), dt_softplus=True, return_state=True)
    ref.check(got, y, bound)
    ref.check(last, end, end_bound, "state")


def test_scan_without_frames_keeps_the_state(seq):
    s = rand(53, 2, 6, 5).cuda()
    d = on_gpu(scan_inputs(54, 2, 1, 6, 5, 1, F32))
    d = {k: v if k in ("A", "D", "dt_bias") else v[:, :0] for k, v in d.items()}
    y, end = seq.selective_scan(**d, state=s, return_state=True)
    assert y.shape == (2, 0, 6) and torch.equal(end, s)
    y, end = seq.selective_scan(**d, return_state=True)
    assert not bool(end.any())


# ------------------------------------------------------------------------------------------------------------- together
def layer_weights(c, m, k):
    return dict(norm_w=rand(60, c, offset=1.0, scale=0.1).cuda(), norm_b=rand(61, c, scale=0.1).cuda(),
                conv_w=rand(62, c, k, scale=0.5).cuda(), conv_b=rand(63, c, scale=0.1).cuda(),
                A=-torch.exp(rand(64, c, m, scale=0.5)).cuda(), D=rand(65, c).cuda(), dt_bias=rand(66, c, scale=0.3).cuda(),
                to_bc=rand(67, c, 2 * m, scale=c ** -0.5).cuda(), to_dt=rand(68, c, c, scale=c ** -0.5).cuda())


def layer(seq, w, x, lengths=None, reverse=False):
    m = w["A"].shape[1]
    u = seq.group_norm(x, 4, w["norm_w"], w["norm_b"], activation="silu", lengths=lengths)
    v = seq.causal_conv1d(u, w["conv_w"], w["conv_b"], "silu", lengths=lengths, reverse=reverse)
    bc = v @ w["to_bc"]
    return seq.selective_scan(v, v @ w["to_dt"], w["A"], bc[..., :m], bc[..., m:], D=w["D"], z=u, dt_bias=w["dt_bias"],
                              dt_softplus=True, lengths=lengths, reverse=reverse), u


def test_a_layer_of_them_over_clips_and_frame_by_frame(seq):
    c, m, k, n, t = 48, 16, 4, 3, 60
    w, x = layer_weights(c, m, k), rand(69, n, t, c).cuda()
    whole, u = layer(seq, w, x)
    conv_state, scan_state = torch.zeros(n, k - 1, c, device="cuda"), torch.zeros(n, c, m, device="cuda")
    outs = []
    for i in range(t):
        v = seq.causal_conv1d_step(u[:, i], conv_state, w["conv_w"], w["conv_b"], "silu")
        bc = v @ w["to_bc"]
        outs.append(seq.selective_step(v, v @ w["to_dt"], w["A"], bc[:, :m], bc[:, m:], scan_state, D=w["D"], z=u[:, i],
                                       dt_bias=w["dt_bias"], dt_softplus=True))
    torch.testing.assert_close(torch.stack(outs, 1), whole, rtol=1e-4, atol=1e-4)
    # a padded batch gives each clip what it gets alone, in both directions
    lengths = [60, 17, 1]
    for reverse in (False, True):
        padded, _ = layer(seq, w, x, lengths=lengths, reverse=reverse)
        for i, v in enumerate(lengths):
            alone, _ = layer(seq, w, x[i:i + 1, :v], reverse=reverse)
            torch.testing.assert_close(padded[i:i + 1, :v], alone, rtol=1e-4, atol=1e-4)
            assert not bool(padded[i, v:].any())


def test_a_layer_on_another_stream_and_in_a_graph(seq):
    c, m, k, n, t = 32, 8, 3, 2, 1300                              # long enough for runs: a workspace inside the graph
    w, x = layer_weights(c, m, k), rand(70, n, t, c).cuda()
    lengths = torch.tensor([1300, 700]).cuda()
    want, _ = layer(seq, w, x, lengths)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got, _ = layer(seq, w, x, lengths)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):                                             # two captured graphs at once
        held = x.clone()
        with torch.cuda.stream(other):
            layer(seq, w, held, lengths)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = layer(seq, w, held, lengths)
        graphs.append((graph, held, out))
    for i in range(4):
        fresh = rand(71 + i, n, t, c).cuda()
        want, _ = layer(seq, w, fresh, lengths)
        for graph, held, out in graphs:
            held.copy_(fresh)
            graph.replay()
        torch.cuda.synchronize()
        for _, _, out in graphs:
            assert torch.equal(out, want)


def test_captured_steps_move_their_states_on_at_every_replay(seq):
    c, m, k, n = 40, 16, 4, 5
    w = layer_weights(c, m, k)

    def step(x, conv_state, scan_state):
        v = seq.causal_conv1d_step(x, conv_state, w["conv_w"], w["conv_b"], "silu")
        bc = v @ w["to_bc"]
        return seq.selective_step(v, v @ w["to_dt"], w["A"], bc[:, :m], bc[:, m:], scan_state, D=w["D"], z=x,
                                  dt_bias=w["dt_bias"], dt_softplus=True)

    def fresh():
        return torch.zeros(n, k - 1, c, device="cuda"), torch.zeros(n, c, m, device="cuda")

    held, states, eager = torch.zeros(n, c, device="cuda"), fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, *fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, *states)
    for i in range(6):
        x = rand(100 + i, n, c).cuda()
        want = step(x, *eager)
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(states[0], eager[0]) and torch.equal(states[1], eager[1])


def test_kernels_report_to_the_profiler(seq):
    from sound_event_detection_amd import _lib
    d = on_gpu(scan_inputs(97, 1, 300, 16, 4, 1, F32))
    _lib.profile_enable(True)
    try:
        seq.group_norm(d["x"], 2)
        seq.causal_conv1d(d["x"], torch.zeros(16, 4, device="cuda"))
        seq.selective_scan(**d, dt_softplus=True)
        names = {k["name"] for k in _lib.profile_collect()}
    finally:
        _lib.profile_enable(False)
    assert {"norm_slab_kernel", "causal_conv_kernel", "selective_scan_end_kernel", "selective_scan_kernel"} <= names


def test_the_same_call_gives_the_same_bits(seq):
    d = on_gpu(scan_inputs(80, 1, 1500, 40, 16, 1, BF16))
    x = rand(81, 2, 500, 16, 64).cuda()
    first = seq.selective_scan(**d, dt_softplus=True), seq.group_norm(x, 8)
    for _ in range(3):
        assert torch.equal(seq.selective_scan(**d, dt_softplus=True), first[0])
        assert torch.equal(seq.group_norm(x, 8), first[1])


def test_offsets_beyond_32_bits(seq):
    c, m = 16, 4
    buf = torch.zeros(5 << 30, dtype=F16, device="cuda")            # 10 GiB: clips and frames far apart in it
    far = (1 << 31) + 4096
    lead = dict(size=(2, 40, c), stride=(far, 1 << 25, 1))          # frames 2^25 elements apart, clips 2^31
    x = buf.as_strided(**lead)
    x.copy_(rand(90, 2, 40, c, dtype=F16))
    d = scan_inputs(91, 2, 40, c, m, 1, F16)
    d["x"] = x.cpu().contiguous()
    y, bound, _, _ = ref.selective_scan(**d, dt_softplus=True)
    ref.check(seq.selective_scan(**{**on_gpu(d), "x": x}, dt_softplus=True), y, bound)
    w = rand(92, c, 4)
    y, bound, _ = ref.causal_conv1d(d["x"], w)
    ref.check(seq.causal_conv1d(x, w.cuda()), y, bound)
    del x, buf
    big = torch.zeros((3, (1 << 20) + 3, 1, 1024), dtype=F16, device="cuda")      # over 2^31 elements, contiguous
    big[2, -1, 0] = rand(93, 1024, dtype=F16).cuda()
    got = seq.group_norm(big, 1)
    row = big[2, -1, 0].double()
    count = big[2].numel()
    mean, var = row.sum() / count, (row ** 2).sum() / count - (row.sum() / count) ** 2
    want = (row - mean) / torch.sqrt(var + 1e-5)
    assert float((got[2, -1, 0].double() - want).abs().max()) <= 2.0 ** -11 * float(want.abs().max()) * 1.1
    assert not bool(got[:2].any())


# ------------------------------------------------------------------------------------------------------------- refusals
def test_refusals(seq):
    from sound_event_detection_amd import _lib
    x = torch.zeros(2, 5, 8, device="cuda")
    w = torch.zeros(8, 4, device="cuda")
    d = on_gpu(scan_inputs(95, 2, 5, 8, 4, 1, F32))
    for call in (lambda: seq.group_norm(x.cpu(), 2), lambda: seq.causal_conv1d(x.cpu(), w.cpu()),
                 lambda: seq.selective_scan(**{**d, "x": x.cpu()})):
        with pytest.raises(_lib.SedmiError):
            call()
    for call in (lambda: seq.group_norm(x, 3), lambda: seq.group_norm(x, 0), lambda: seq.group_norm(x, 2, activation="tanh"),
                 lambda: seq.group_norm(x, 2, eps=-1.0), lambda: seq.group_norm(x, 2, torch.zeros(7, device="cuda")),
                 lambda: seq.group_norm(x, 2, lengths=[1]), lambda: seq.group_norm(x[:, 0], 2, lengths=[1, 1]),
                 lambda: seq.causal_conv1d(x, torch.zeros(8, 9, device="cuda")),
                 lambda: seq.causal_conv1d(x, torch.zeros(7, 4, device="cuda")),
                 lambda: seq.causal_conv1d(x, w, state=torch.zeros(2, 4, 8, device="cuda")),
                 lambda: seq.causal_conv1d(x[0], w), lambda: seq.causal_conv1d(x, w, lengths=[5, 5, 5]),
                 lambda: seq.causal_conv1d_step(x[:, 0], torch.zeros(2, 8, 3, device="cuda").transpose(1, 2), w),
                 lambda: seq.selective_scan(**{**d, "dt": d["dt"][:, :4]}),
                 lambda: seq.selective_scan(**{**d, "A": torch.zeros(8, 129, device="cuda")}),
                 lambda: seq.selective_scan(**{**d, "B": d["B"][..., :3]}),
                 lambda: seq.selective_scan(**{**d, "B": d["B"].expand(2, 5, 3, 4), "C": d["C"].expand(2, 5, 3, 4)}),
                 lambda: seq.selective_scan(**d, state=torch.zeros(2, 8, 5, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: seq.group_norm(x.double(), 2), lambda: seq.group_norm(x, 2, lengths=torch.tensor([1.0, 2.0])),
                 lambda: seq.group_norm(x, 2, torch.zeros(8)), lambda: seq.causal_conv1d(x, w.cpu()),
                 lambda: seq.causal_conv1d(x, w, state=torch.zeros(2, 3, 8, device="cuda", dtype=F16)),
                 lambda: seq.selective_scan(**{**d, "z": d["z"].half()}),
                 lambda: seq.selective_scan(**d, state=torch.zeros(2, 8, 4, device="cuda", dtype=F16))):
        with pytest.raises(TypeError):
            call()
    one = {k: v if k in ("A", "D", "dt_bias") else v[:, 0] for k, v in d.items()}
    with pytest.raises(ValueError):
        seq.selective_step(**one, state=torch.zeros(2, 8, 4, device="cuda", dtype=F16))
    with pytest.raises(ValueError):
        seq.selective_step(**one, state=torch.zeros(2, 4, 8, device="cuda").transpose(1, 2))
    with pytest.raises(RuntimeError, match="inference-only"):
        seq.group_norm(x.requires_grad_(), 2)
    with torch.no_grad():
        assert seq.group_norm(x, 2).shape == x.shape
