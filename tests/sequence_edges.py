"""Group norm in float64 over all groups at once, with the error of the kernels' own order of summation, for shapes at which
the bound of sequence_reference.py (one addition per row, whatever the kernel) says too little or takes too long."""
import torch

import sequence_reference as ref
from sequence_reference import U

THREADS = 256


def two_launch_depth(clips, rows, channels, groups, dtype):
    """(chunks, depth): the row chunks of the two-launch form and how many roundings of the size of the mean an element
    passes there: half the rows of a thread (step k of the running mean is off by U |mean| and counts k / n of the result),
    the channels of a vector, the entries a wave's lane walks, 6 shuffles, then 4 chunks of a lane and 6 shuffles, and the
    divisions."""
    vec = 4 if dtype == torch.float32 else 8
    per = channels // groups
    most_groups = max(1, min(groups, THREADS * vec // per))
    blocks = -(-groups // most_groups)
    vectors = min(THREADS, -(-(-(-groups // blocks) * per) // vec))
    lanes = THREADS // vectors
    chunks = max(1, min(-(-512 // max(1, clips * blocks)), max(1, rows // (lanes * 4)), 256))
    each = -(-(-(-rows // chunks)) // lanes)
    turns = -(-(-(-per // vec)) // THREADS)                     # columns of a thread, of a group wider than a workgroup
    joined = -(-groups // blocks) == 1 or per % vec == 0         # a thread's channels lie in one group: one entry of it
    walk = THREADS // 64 if joined else -(-lanes * per // 64)
    return chunks, each / 2 + vec + 2 * turns + walk + 6 + 4 + 6 + 6


def one_launch_depth(rows, channels, groups, dtype):
    """(vectors of a thread, depth): the elements a thread adds up, 6 shuffles, 16 waves, a division."""
    vec = 4 if dtype == torch.float32 else 8
    vectors = rows * -(-(channels // groups) // vec)
    threads = 256 if vectors <= 512 else 512 if vectors <= 1024 else 1024
    each = -(-vectors // threads)
    return each, each * vec + 6 + 16 + 2


def group_norm(x, groups, weight, bias, eps, depth, activation=None, lengths=None):
    """(y, bound).  x [clips, frames, inner, channels].

    The mean is off by e = U (depth (|m| + s) + 3 max|x - m|), s the standard deviation: depth roundings of values around
    the mean, and the running mean's steps, each 3 U of a deviation over its number.  The squares: U each (depth + 40) times
    of their sum, and the mean's error twice in each deviation, 4 e s + 4 e^2.  The rest as in sequence_reference.py."""
    n, frames, inner, c = x.shape
    y, bound = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    w, b = weight.double(), bias.double()
    for i, t in enumerate(ref.valid_frames(lengths, n, frames)):
        if t == 0:
            continue
        part = x[i, :t].double().reshape(t * inner, groups, c // groups)
        m = part.mean((0, 2), keepdim=True)
        off = part - m
        v = (off * off).mean((0, 2), keepdim=True)
        e = U * (depth * (m.abs() + v.sqrt()) + 3 * off.abs().amax((0, 2), keepdim=True))
        dv = U * (depth + 40) * v + 4 * e * v.sqrt() + 4 * e * e
        half = 0.5 * dv / (v + eps)
        dr = half + 2 * half * half + 4 * U
        r = 1 / torch.sqrt(v + eps)
        shape = (t, inner, c)
        normal = (off * r).reshape(shape)
        s = normal * w + b
        err = w.abs() * (r * (e + U * off.abs()) + (off * r).abs() * (dr + 4 * U)).reshape(shape) + U * s.abs()
        y[i, :t] = ref.act(s, activation)
        bound[i, :t] = ref.act_bound(s, y[i, :t], err, activation)
    return y, bound


# Groups of few channels, groups that end inside a vector, a group of whole vectors and one wider than a workgroup; the last
# has one chunk per clip and long columns.
FAR_SHAPES = [(2, 1500, 1, 24, 12), (2, 2500, 1, 60, 10), (2, 1200, 4, 16, 2), (2, 70, 1, 5000, 1), (512, 640, 1, 30, 10)]


def far_input(shape):
    """Mean 500, deviation 0.25: plain float32 sums of squares keep no digit of the variance."""
    n, t, inner, c, groups = shape
    g = torch.Generator().manual_seed(200)
    x = torch.randn(n, t, inner, c, generator=g) * 0.25 + 500
    return x, torch.rand(c, generator=g) + 0.5, torch.randn(c, generator=g)
