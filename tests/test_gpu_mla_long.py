"""GPU: absorbed attention where a CTA pair walks over several tiles of a unit,
so that the running reference of the softmax is raised inside a piece, and the
pieces that pairs leave of one unit are joined: against the plain 64-bit form
of tests/mla_ref.py."""
import numpy as np
import pytest

import mla_ref as R
from test_gpu_mla import Paged, m, run_attend  # noqa: F401  (m: the context fixture)

pytestmark = pytest.mark.gpu
TILE, RAISE = 64, 8.0   # cache rows of a tile; log2 by which scores may pass the reference
LN2 = float(np.log(2.0))


def pairs():
    import torch
    return torch.cuda.get_device_properties(0).multi_processor_count // 2


def tiles_per_pair(lens, heads):
    return sum(-(-n * heads // 128) * -(-(c + n) // TILE) for c, n in lens) / pairs()


def bounds(want, wl, A, S, t, tiles):
    """R.attend_bounds, whose 2^-20 of A stands for few tiles: the output's sums of a piece take 4 steps a tile, each
    cut to fp32 at most once, the join one more per piece; sums of weights the same."""
    tol, tl = R.attend_bounds(want, wl, A, S, t)
    steps = (4 * tiles + pairs()) * 2.0 ** -23
    return tol + steps * A, tl + steps


def check(g, q, scale, out, lse, tiles):
    t = R.kind(g.fmt)
    qv = R.rounded(q, t)
    for b, (c, n) in enumerate(g.lens):
        s = slice(g.start[b], g.start[b + 1])
        kv = R.unpack(g.host[g.rows(b, 0, c + n)], g.latent, g.fmt)
        vis = np.concatenate([np.ones((n, c), bool), np.tril(np.ones((n, n), bool))], 1)
        want, wl, A, S = R.attend(qv[s], kv, vis, scale, g.latent)
        tol, tl = bounds(want, wl, A, S, t, tiles)
        bad = ~(np.abs(out[s] - want) <= tol)
        assert not bad.any(), (b, bad.sum(), np.argwhere(bad)[:4], out[s][bad][:4], want[bad][:4], tol[bad][:4])
        assert np.all(np.abs(lse[s] - wl) <= tl), (b, np.max(np.abs(lse[s] - wl) - tl))


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("latent", [512, 128])
def test_halves_whose_references_part(m, cuda_lib, fmt, latent):  # noqa: F811
    """The two CTAs of a pair sum a score's halves in different orders.  Here the halves are large and cancel, so the
    two scores differ in their last bits; one row of a piece lies at the reference + 8 log2 up to those bits, so
    that often one of the CTAs raises its reference there and the other does not."""
    n_rows = 9 * pairs() * TILE - 40
    g = Paged(cuda_lib, [(n_rows - 1, 1)], fmt, latent, 64)
    assert tiles_per_pair(g.lens, 128) > 8
    rng = np.random.default_rng(latent)
    half = np.abs(rng.standard_normal((n_rows, latent // 2))) * 4
    # scores in log2: the reference's row of each tile 0, the others far below it, one row of every ninth tile + 8
    target = np.full(n_rows, -10.0)
    target[::TILE] = 0.0
    target[4 * TILE + 5::9 * TILE] = RAISE
    rope = np.zeros((n_rows, 64))
    rope[:, 0] = target
    # page by page: the rows are many
    g.host[g.rows(0, 0, n_rows)] = R.pack(np.concatenate([half, half], 1).astype(np.float32), rope.astype(np.float32), fmt)
    g.upload()
    q = np.zeros((1, 128, latent + 64))
    side = np.repeat(np.abs(rng.standard_normal((4, latent // 2))), 32, 0)   # a warp's 32 rows alike
    q[0, :, :latent // 2], q[0, :, latent // 2:latent] = side, -side
    q[0, :, latent] = 1.0
    out, lse = run_attend(m, g, q, LN2, R.kind(fmt))
    check(g, q, LN2, out, lse, 10)
    # rows hold the same values in both halves, so both halves of the output are the same up to their errors
    assert np.allclose(out[..., :latent // 2], out[..., latent // 2:], rtol=0.1)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("shape", ["cut", "whole", "both"])
def test_reference_raised_inside_a_piece(m, cuda_lib, fmt, shape):  # noqa: F811
    """Scores that climb by more than 8 log2 from tile to tile inside a piece, fall back, and climb by less: units cut
    into pieces of many tiles, whole units of several tiles, and both at once."""
    p = pairs()
    lens = {"cut": [(8 * p * TILE + 17, 1)], "whole": [(6 * TILE - 1 - (b % 3), 1) for b in range(2 * p)],
            "both": [(5 * TILE + 3, 2)] * p + [(2 * p * TILE, 1)]}[shape]
    heads = 128
    assert tiles_per_pair(lens, heads) > 7
    g = Paged(cuda_lib, lens, fmt, 128, 64, seed=1)
    rng = np.random.default_rng(len(lens))
    # the climb inside any 3 tiles passes 8 log2 for some heads (head h turns the climb by its own factor)
    level = np.array([0.0, 6.0, 20.0, 3.0, 33.0, 34.0, -5.0, 60.0])
    for b, (c, n) in enumerate(lens):
        r = c + n
        lat = rng.standard_normal((r, 128)).astype(np.float32) * 0.25
        rope = np.zeros((r, 64), np.float32)
        rope[:, 0] = level[(np.arange(r) // TILE + b) % len(level)]
        rope[:, 1] = 0.5 * rng.standard_normal(r)
        g.host[g.rows(b, 0, r)] = R.pack(lat, rope, fmt)
    g.upload()
    q = rng.standard_normal((g.T, heads, 192)) * 0.25
    q[..., 128:] = 0
    q[..., 128] = np.linspace(-1, 1, heads)
    q[..., 129] = 1.0
    out, lse = run_attend(m, g, q, LN2, R.kind(fmt))
    check(g, q, LN2, out, lse, 10)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("below", [8.0, 13.0, 16.0, 17.2, 17.35, 19.0])
def test_a_strong_first_row_does_not_hide_the_tail(m, cuda_lib, fmt, below):  # noqa: F811
    """One row (of value 0) takes most of the weight in front of 131,071 rows (of value 1), `below` nats lower."""
    n_rows, latent = 131072, 128
    g = Paged(cuda_lib, [(n_rows - 1, 1)], fmt, latent, 64, seed=2)
    lat = np.ones((n_rows, latent), np.float32)
    lat[0] = 0
    rope = np.zeros((n_rows, 64), np.float32)
    rope[0, 0] = 1
    g.host[g.rows(0, 0, n_rows)] = R.pack(lat, rope, fmt)
    g.upload()
    q = np.zeros((1, 16, latent + 64))
    q[..., latent] = np.linspace(0.9, 1.0, 16) * 64
    scale = below / 64
    t = R.kind(fmt)
    out, lse = run_attend(m, g, q, scale, t)
    # in closed form (the rows are two kinds): weights 1 and e^-s, s the strong row's score
    s = scale * R.rounded(q, t)[0, :, latent]
    tail = (n_rows - 1) * np.exp(-s)
    want = tail / (1 + tail)
    # as R.attend_bounds, and what fp16 adds: a weight of at least 2^-32 of the reference's keeps an error of at most
    # that, for each row, where it is below fp16's normal range; then the sums' steps
    tol, tl = bounds(want[:, None], s + np.log1p(tail), want[:, None], s, t, -(-n_rows // TILE) / pairs() + 1)
    if t == "f16":
        tol = tol + (n_rows * 2.0 ** -32 / (1 + tail))[:, None]
    assert np.all(np.abs(out[0] - want[:, None]) <= tol), (out[0, :, 0], want, tol[:, 0])
    assert np.all(np.abs(lse[0] - s - np.log1p(tail)) <= tl)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 23, 2.0 ** 25])
def test_huge_scores_stay_finite(m, cuda_lib, fmt, size):  # noqa: F811
    """Scores (in log2, up to twice `size`) whose own rounding is up to 4: the strongest row wins, nothing overflows."""
    p = pairs()
    n_rows = 8 * p * TILE
    g = Paged(cuda_lib, [(n_rows - 1, 1)], fmt, 128, 64, seed=3)
    rng = np.random.default_rng(1)
    lat = rng.standard_normal((n_rows, 128)).astype(np.float32)
    rope = np.zeros((n_rows, 64), np.float32)
    rope[:, 0] = rng.uniform(0.5, 1.0, n_rows)
    rope[n_rows // 3 + 7, 0] = 2.0
    g.host[g.rows(0, 0, n_rows)] = R.pack(lat, rope, fmt)
    g.upload()
    q = np.zeros((1, 128, 192))
    q[..., 128] = np.linspace(0.5, 1.0, 128)
    scale = size * LN2
    out, lse = run_attend(m, g, q, scale, R.kind(fmt))
    row = R.unpack(g.host[g.rows(0, n_rows // 3 + 7, n_rows // 3 + 8)], 128, fmt)[0, :128]
    want = np.broadcast_to(row, (128, 128))
    s = scale * R.rounded(q, R.kind(fmt))[0, :, 128] * 2.0
    assert np.all(np.abs(out[0] - want) <= 2 * R.U[R.kind(fmt)] * np.abs(want) * 1.01)
    assert np.all(np.abs(lse[0] - s) <= 2.0 ** -20 * s)
