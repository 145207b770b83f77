"""GPU: rotary positions, the paged latent cache (write, read) and the absorbed
attention of drafted tokens, through the C ABI, each against a plain 64-bit
form (tests/mla_ref.py) at the sizes, masks and layouts where it can go wrong;
and the operators together as a decode step uses them, against the oracle's
mla_forward."""
import numpy as np
import pytest

import mla_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": 0, "f16": 1, "bf16": 30}


@pytest.fixture(scope="module")
def m(cuda_lib):
    ctx = cuda_lib.MoE(cuda_lib.MoeConfig(hidden=256, intermediate=256, n_experts=8, n_group=2, topk_group=1, top_k=2,
                                          max_tokens=1))
    yield ctx
    ctx.close()


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ready(m):
    """The library runs on its own stream: inputs first, results after."""
    import torch
    torch.cuda.synchronize()


def typed(x, t):
    """Host values as the bytes of type t, and the values they hold."""
    x = np.asarray(x, np.float32)
    if t == "f32":
        return x, x.astype(np.float64)
    return R.to_bits(x, t), R.from_bits(R.to_bits(x, t), t)


def back(d, t):
    a = d.cpu().numpy()
    return a.astype(np.float64) if t == "f32" else R.from_bits(a.view(np.uint16), t)


# ------------------------------------------------------------------- rotary
@pytest.mark.parametrize("ti,to", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"),
                                   ("f16", "bf16")])
@pytest.mark.parametrize("T,H,D,off,dim,half", [(1, 128, 64, 0, 64, False), (3, 5, 192, 128, 64, False),
                                                (7, 3, 80, 0, 80, True), (2, 1, 10, 3, 6, False), (5, 2, 37, 1, 36, True),
                                                (4, 9, 256, 0, 256, True), (1, 1, 2, 0, 2, False),
                                                (2, 3, 24, 8, 8, False), (2, 3, 24, 8, 8, True)])
def test_rope(m, cuda_lib, ti, to, T, H, D, off, dim, half):
    import torch
    rng = np.random.default_rng(T * 1000 + D)
    raw, x = typed(rng.standard_normal((T, H, D)), ti)
    pos = rng.integers(-50, 1 << 20, T).astype(np.int32)
    pos[0] = 0 if T > 1 else (1 << 31) - 1
    cfg = cuda_lib.RopeConfig(dim=dim, half_layout=half, mscale=1.25)
    d = dev(raw)
    y = torch.zeros((T, H, D), dtype=torch.float32 if to == "f32" else torch.int16, device="cuda")
    p = dev(pos)
    ready(m)
    m.rope_device(cfg, d, DT[ti], (H * D, D), y, DT[to], (H * D, D), p, T, H, D, off)
    m.check_error()
    f = R.freqs(dim)
    want = x.copy()
    want[..., off:off + dim] = R.rotate(x[..., off:off + dim], pos, f, half, 1.25)
    # cos and sin: the reduced angle rounded to fp32 (2^-25 of a turn), sincospi's 2 ulp, mscale: under 2^-21
    # together; two products and a sum: 3 * 2^-24; then one rounding to the result's type
    pair = np.abs(x[..., off:off + dim])
    partner = np.concatenate([pair[..., dim // 2:], pair[..., :dim // 2]], -1) if half else \
        pair.reshape(T, H, -1, 2)[..., ::-1].reshape(pair.shape)
    tol = R.U[to] * np.abs(want) + 2.0 ** -24 * (to == "f16")
    # the turns themselves in 64 bits: pos * 2^-52 turns
    tol[..., off:off + dim] += 1.25 * (pair + partner) * (1.01 * 2.0 ** -20.5 + 8 * np.abs(pos.astype(np.float64))[:, None, None] * 2.0 ** -52)
    assert np.all(np.abs(back(y, to) - want) <= tol)


@pytest.mark.parametrize("half", [False, True])
def test_rope_strides_and_in_place(m, cuda_lib, half):
    """Heads in front of tokens, unaligned rows, a broadcast input; in place leaves the other values alone."""
    import torch
    rng = np.random.default_rng(5)
    T, H, D, off, dim = 4, 3, 72, 8, 64
    x = rng.standard_normal((H, T, D + 1)).astype(np.float32)
    pos = np.array([9, 0, 77777, 5], np.int32)
    cfg = cuda_lib.RopeConfig(dim=dim, half_layout=half, scale=1.0)
    d, p = dev(x), dev(pos)
    y = torch.full((T, H, D + 3), 7.0, device="cuda")
    ready(m)
    m.rope_device(cfg, d, 0, (D + 1, T * (D + 1)), y, 0, (H * (D + 3), D + 3), p, T, H, D, off)
    m.check_error()
    want = x.transpose(1, 0, 2)[..., :D].astype(np.float64)
    want[..., off:off + dim] = R.rotate(want[..., off:off + dim].copy(), pos, R.freqs(dim, scale=1.0), half)
    got = y.cpu().numpy()
    assert np.max(np.abs(got[..., :D] - want)) < 8 * 2.0 ** -21 and np.all(got[..., D:] == 7.0)
    m.rope_device(cfg, d, 0, (D + 1, T * (D + 1)), d, 0, (D + 1, T * (D + 1)), p, T, H, D, off)
    m.check_error()
    assert np.array_equal(d.cpu().numpy().transpose(1, 0, 2)[..., :D], got[..., :D])
    assert np.array_equal(d.cpu().numpy()[..., D], x[..., D])
    one = dev(x[:1, :1, :D])
    m.rope_device(cfg, one, 0, (0, 0), y, 0, (H * (D + 3), D + 3), p, T, H, D, off)
    m.check_error()
    b = np.broadcast_to(x[0, 0, :D].astype(np.float64), (T, H, D)).copy()
    b[..., off:off + dim] = R.rotate(b[..., off:off + dim].copy(), pos, R.freqs(dim, scale=1.0), half)
    assert np.max(np.abs(y.cpu().numpy()[..., :D] - b)) < 8 * 2.0 ** -21


# -------------------------------------------------------------------- cache
class Paged:
    """A cache of `lens` = [(rows before the call, rows of the call)] with shuffled pages; `fill` rows' bytes."""

    def __init__(self, F, lens, fmt, latent, page, seed=0, extra=2, q0=0, fill=255):
        import torch
        rng = np.random.default_rng(seed)
        self.F, self.lens, self.fmt, self.latent, self.page = F, lens, fmt, latent, page
        need = [-(-(c + n) // page) for c, n in lens]
        self.per = max(need + [1])
        self.n_pages = sum(need) + extra
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.per), -1, np.int32)   # entries past a sequence's end are never looked at
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.start = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32) + q0
        self.ctx = np.array([c for c, _ in lens], np.int32)
        self.T = int(self.start[-1])
        # unused rows hold NaN patterns
        self.host = np.full((self.n_pages * page, R.row_bytes(fmt, latent)), fill, np.uint8)
        self.d = torch.zeros(self.host.shape, dtype=torch.uint8, device="cuda")
        self.bufs = [dev(self.start), dev(self.ctx), dev(self.table)]
        self.kv = F.KVCache(self.d, fmt, latent, page, self.n_pages)

    def rows(self, b, lo, hi):
        r = np.arange(lo, hi)
        return self.table[b, r // self.page].astype(np.int64) * self.page + r % self.page

    def batch(self, T=None):
        return self.F.KVBatch(len(self.lens), self.T if T is None else T, *self.bufs, self.per)

    def upload(self):
        import torch
        self.d.copy_(torch.from_numpy(self.host))


LENS = [[(0, 1)], [(5, 1), (0, 0), (63, 2), (8, 17)], [(1000, 3), (0, 64)]]


@pytest.mark.parametrize("lens", LENS, ids=["one", "ragged", "long"])
@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("latent,page,t", [(512, 64, "f32"), (128, 8, "f16"), (384, 16, "bf16"), (256, 128, "f32")])
def test_write_and_read_without_norm_is_exact(m, cuda_lib, lens, fmt, latent, page, t):
    """Stored bytes equal the format's definition; what is read back equals what the bytes stand for."""
    import torch
    g = Paged(cuda_lib, lens, fmt, latent, page)
    rng = np.random.default_rng(latent + fmt)
    T, W = g.T, latent + 64
    vals = rng.standard_normal((T + 1, W)) * 10.0 ** rng.integers(-6, 5, (T + 1, 1))
    vals[0, :32] = 0
    raw, x = typed(vals, t)
    g.upload()
    before = g.d.cpu().numpy()
    d = dev(raw)
    ready(m)
    # one row more than the sequences hold: it belongs to none
    m.kv_write_device(g.kv, g.batch(T + 1), d, DT[t], W)
    m.check_error()
    want = before.copy()
    used = latent + 128 + latent // 32 if R.is_fp8(fmt) else want.shape[1]
    for b, (c, n) in enumerate(lens):
        at = g.rows(b, c, c + n)
        sl = slice(g.start[b], g.start[b + 1])
        want[at, :used] = R.pack(x[sl, :latent], x[sl, latent:], fmt)[:, :used]
    got = g.d.cpu().numpy()
    assert np.array_equal(got[:, :used], want[:, :used])
    for to in ("f32", R.kind(fmt)):
        y = torch.full((T + 1, W), 77, dtype=torch.float32 if to == "f32" else torch.int16, device="cuda")
        ready(m)
        m.kv_read_device(g.kv, g.batch(T + 1), y, DT[to], W)
        m.check_error()
        a = back(y, to)
        for b, (c, n) in enumerate(lens):
            assert np.array_equal(a[g.start[b]:g.start[b + 1]], R.unpack(got[g.rows(b, c, c + n)], latent, fmt), equal_nan=True)
        assert np.all(y[T].cpu().numpy() == 77)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("latent,t,half", [(512, "f32", False), (512, "bf16", False), (128, "f16", True), (384, "f32", True)])
def test_write_norm_and_rope(m, cuda_lib, fmt, latent, t, half):
    lens = [(3, 9), (70, 30)]
    g = Paged(cuda_lib, lens, fmt, latent, 16)
    rng = np.random.default_rng(latent)
    raw, x = typed(rng.standard_normal((g.T, latent + 67)) * 2, t)    # rows 67 - 64 values apart: not on 16 bytes
    w = (1 + 0.2 * rng.standard_normal(latent)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, g.T).astype(np.int32)
    d, dw, dp = dev(raw), dev(w), dev(pos)
    ready(m)
    m.kv_write_device(g.kv, g.batch(), d, DT[t], latent + 67, dw, 1e-6, cuda_lib.RopeConfig(half_layout=half), dp)
    m.check_error()
    lat = R.rmsnorm(x[:, :latent], w, 1e-6)
    rope = R.rotate(x[:, latent:latent + 64], pos, R.freqs(), half)
    got = g.d.cpu().numpy()
    at = np.concatenate([g.rows(b, c, c + n) for b, (c, n) in enumerate(lens)])
    v = R.unpack(got[at], latent, fmt)
    u = R.U[R.kind(fmt)]
    # the norm in fp32: 16 + 5 additions, a division, a root, three products: under 2^-18 relative
    near = 2.0 ** -18 * np.abs(lat)
    if R.is_fp8(fmt):   # half a step of e4m3 (2^-4), or of its smallest steps (2^-10 of the group's scale)
        sc = np.repeat(2.0 ** (got[at][:, latent + 128:latent + 128 + latent // 32].astype(np.float64) - 127), 32, 1)
        near += np.maximum(2.0 ** -4 * np.abs(lat), 2.0 ** -10 * sc)
        big = np.max(np.abs(lat).reshape(g.T, -1, 32), -1)
        fit = 448.0 * sc[:, ::32]
        assert np.all(big <= fit * (1 + 2.0 ** -18)) and np.all(big >= fit / 2 * (1 - 2.0 ** -18))
    else:
        near += u * np.abs(lat)
    assert np.all(np.abs(v[:, :latent] - lat) <= near * 1.01)
    far = np.repeat(np.abs(x[:, latent:latent + 64]).max(1, keepdims=True), 64, 1)
    assert np.all(np.abs(v[:, latent:] - rope) <= u * np.abs(rope) + far * 2.0 ** -19 + 2.0 ** -24)


@pytest.mark.parametrize("fmt", [R.FP8_BF16, R.FP8_F16])
def test_write_extremes(m, cuda_lib, fmt):
    """Infinities and NaN poison their group alone; huge values saturate; denormals, zeros and ties round as defined."""
    g = Paged(cuda_lib, [(0, 8)], fmt, 128, 8)
    x = np.ones((8, 192), np.float32)
    x[0, 3], x[1, 40] = np.inf, np.nan
    x[2, :32] = 1e30
    x[3, :32] = 1e-42
    x[4, :32] = np.float32(448.0)
    x[4, 0] = np.float32(448.0) * np.float32(1 + 2.0 ** -23)
    x[5, :32] = np.arange(32) * 0.0625 + 17 / 16    # ties of e4m3 among them
    x[6, :32] = -0.0
    d = dev(x)
    ready(m)
    m.kv_write_device(g.kv, g.batch(), d, 0, 192)
    m.check_error()
    want = R.pack(x[:, :128].astype(np.float64), x[:, 128:], fmt)
    got = g.d.cpu().numpy()[g.rows(0, 0, 8)]
    assert np.array_equal(got[:, 256:260], want[:, 256:260])
    assert got[0, 256] == 255 and got[0, 257] != 255 and got[1, 257] == 255
    ok = np.repeat(want[:, 256:260] != 255, 32, 1)
    assert np.array_equal(got[:, :128][ok], want[:, :128][ok])
    v = R.unpack(got, 128, fmt)
    assert np.all(np.isnan(v[0, :32])) and not np.any(np.isnan(v[0, 32:])) and np.all(v[2, :32] == 57344)


def test_bad_pages_and_bounds_are_reported(m, cuda_lib):
    """Rows without a valid page are skipped by the write, read as zeros, seen by nobody; the context says so."""
    import torch
    F = cuda_lib
    lens = [(0, 8), (3, 8)]
    g = Paged(F, lens, R.BF16, 128, 8)
    g.table[1, 1] = 10 ** 6
    g.bufs[2] = dev(g.table)
    raw, x = typed(np.random.default_rng(1).standard_normal((16, 192)), "f32")
    d = dev(raw)
    ready(m)
    m.kv_write_device(g.kv, g.batch(), d, 0, 192)
    with pytest.raises(F.MoeError, match="page"):
        m.check_error()
    m.check_error()   # cleared
    y = torch.full((16, 192), 5.0, device="cuda")
    ready(m)
    m.kv_read_device(g.kv, g.batch(), y, 0, 192)
    with pytest.raises(F.MoeError, match="page"):
        m.check_error()
    got = y.cpu().numpy()
    assert np.array_equal(got[:13], R.rounded(x[:13], "bf16").astype(np.float32)) and np.all(got[13:] == 0)
    # positions outside the table: a context longer than the table, a negative one
    for ctx in (10 ** 9, -5, (1 << 31) - 4):
        g.bufs[1] = dev(np.array([0, ctx], np.int32))
        ready(m)
        m.kv_write_device(g.kv, g.batch(), d, 0, 192)
        with pytest.raises(F.MoeError, match="page"):
            m.check_error()
    g.bufs[1] = dev(g.ctx)
    # the attention: sequence 0 is right, sequence 1 sees its valid rows only
    h, W = 3, 192
    q = np.random.default_rng(2).standard_normal((16, h, W))
    out, lse = run_attend(m, g, q, 0.1, "bf16", check=False)
    with pytest.raises(F.MoeError, match="page"):
        m.check_error()
    qv = R.rounded(q, "bf16")
    kv0 = R.unpack(g.d.cpu().numpy()[g.rows(0, 0, 8)], 128, R.BF16)
    want, wl, A, S = R.attend(qv[:8], kv0, np.tril(np.ones((8, 8), bool)), 0.1, 128)
    tol, tl = R.attend_bounds(want, wl, A, S, "bf16")
    assert np.all(np.abs(out[:8] - want) <= tol) and np.all(np.abs(lse[:8] - wl) <= tl)
    assert np.all(np.isfinite(out))


# ---------------------------------------------------------------- attention
def pack_tree(sees, words):
    """Bool [tokens, drafted rows] -> uint32 [tokens, words]."""
    T, n = sees.shape
    bits = np.zeros((T, words * 32), np.uint8)
    bits[:, :n] = sees
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def run_attend(m, g, q, scale, t, tree=None, pad=0, head_major=False, lse=True, stream=None, ws=None, check=True, batch=None):
    """Queries [tokens, heads, latent + 64] through the library; outputs of rows outside the sequences stay at 7."""
    import torch
    T, h, W = q.shape
    L = W - 64
    ql, qr = np.zeros((T, h, L + 8 * pad), np.float32), np.zeros((T, h, 64 + 8 * pad), np.float32)
    ql[..., :L], qr[..., :64] = q[..., :L], q[..., L:]
    if head_major:
        ql, qr = ql.transpose(1, 0, 2), qr.transpose(1, 0, 2)
    dl, dr = dev(typed(ql, t)[0]), dev(typed(qr, t)[0])
    st = (lambda w: (w, T * w)) if head_major else (lambda w: (h * w, w))
    seven = int(np.array(typed([7.0], t)[0]).view(np.int16)[0])
    shape = (h, T, L + 8 * pad) if head_major else (T, h, L + 8 * pad)
    out = torch.full(shape, seven, dtype=torch.int16, device="cuda")
    d_lse = torch.full((T, h), 7.0, device="cuda") if lse else None
    if ws is None:
        ws = torch.full((m.mla_workspace_bytes(L),), 255, dtype=torch.uint8, device="cuda")
    dt = None if tree is None else dev(tree.view(np.int32))
    ready(m)
    m.mla_attention_device(g.kv, batch or g.batch(), dl, st(L + 8 * pad), dr, st(64 + 8 * pad), h, scale, out, st(L + 8 * pad),
                           ws, ws.numel(), lse=d_lse, tree=dt, tree_words=0 if tree is None else tree.shape[1], stream=stream)
    ready(m)
    if check:
        m.check_error()
    o = back(out, t)
    if head_major:
        o = o.transpose(1, 0, 2)
    assert np.all(o[..., L:] == 7.0)
    return o[..., :L], None if d_lse is None else d_lse.cpu().numpy().astype(np.float64)


def fill(g, seed=0, sigma=1.0):
    """Every row of every sequence; unused rows keep their NaN patterns."""
    rng = np.random.default_rng(seed)
    for b, (c, n) in enumerate(g.lens):
        at = g.rows(b, 0, c + n)
        g.host[at] = R.pack((rng.standard_normal((c + n, g.latent)) * sigma).astype(np.float32),
                            rng.standard_normal((c + n, 64)).astype(np.float32), g.fmt)
    g.upload()


def random_tree(n, rng):
    a = np.zeros((n, n), bool)
    for i in range(n):
        p = rng.integers(-1, i) if i else -1
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def check_attend(g, q, scale, out, lse, sees):
    """sees[b]: [tokens, drafted rows] of sequence b."""
    t = R.kind(g.fmt)
    qv = R.rounded(q, t)
    for b, (c, n) in enumerate(g.lens):
        if not n:
            continue
        s = slice(g.start[b], g.start[b + 1])
        kv = R.unpack(g.host[g.rows(b, 0, c + n)], g.latent, g.fmt)
        vis = np.concatenate([np.ones((n, c), bool), sees[b]], 1)
        want, wl, A, S = R.attend(qv[s], kv, vis, scale, g.latent)
        tol, tl = R.attend_bounds(want, wl, A, S, t)
        bad = ~(np.abs(out[s] - want) <= tol)
        assert not bad.any(), (b, np.argwhere(bad)[:4], np.abs(out[s] - want)[bad][:4], tol[bad][:4])
        if lse is not None:
            empty = np.isneginf(wl)
            assert np.array_equal(np.isneginf(lse[s]), empty)
            assert np.all(np.abs(lse[s] - wl)[~empty] <= tl[~empty])


SHAPES = [
    # (rows before, tokens) of each sequence, heads, latent, page
    ([(0, 1)], 1, 512, 64), ([(1, 1)], 128, 512, 64), ([(62, 1)], 128, 512, 8), ([(63, 1)], 16, 512, 16),
    ([(64, 1)], 128, 512, 128), ([(127, 1), (128, 1), (129, 1)], 5, 512, 32), ([(900, 1)], 128, 512, 64),
    ([(0, 7)], 128, 512, 64), ([(250, 13), (31, 1), (0, 0), (0, 5), (700, 13)], 128, 512, 64),
    ([(100, 5)], 17, 256, 16), ([(33, 3)], 130, 128, 8), ([(200, 70)], 3, 384, 1024), ([(60, 8), (61, 8)], 16, 384, 32),
    ([(5000, 2)], 128, 512, 64), ([(20000, 1)], 16, 512, 64), ([(30, 1)] * 200, 8, 128, 16),
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
@pytest.mark.parametrize("fmt", R.FORMATS)
def test_attend_causal(m, cuda_lib, case, fmt):
    lens, h, latent, page = SHAPES[case]
    g = Paged(cuda_lib, lens, fmt, latent, page, seed=case)
    fill(g, case)
    q = np.random.default_rng(case + 50).standard_normal((g.T, h, latent + 64))
    scale = 2.5 / np.sqrt(latent + 64)
    out, lse = run_attend(m, g, q, scale, R.kind(fmt))
    check_attend(g, q, scale, out, lse, [np.tril(np.ones((n, n), bool)) for _, n in lens])


@pytest.mark.parametrize("fmt", [R.BF16, R.FP8_F16])
@pytest.mark.parametrize("lens,h,words", [([(0, 13)], 128, 1), ([(57, 13), (64, 9), (0, 33)], 16, 2), ([(321, 64)], 5, 3),
                                          ([(63, 2), (1, 100)], 128, 4)])
def test_attend_tree(m, cuda_lib, fmt, lens, h, words):
    """Random trees, extra mask words; drafted rows that a token does not see hold NaN for it in turn."""
    g = Paged(cuda_lib, lens, fmt, 512, 64, seed=3)
    fill(g, 3)
    rng = np.random.default_rng(9)
    sees = [random_tree(n, rng) for _, n in lens]
    tree = np.concatenate([pack_tree(a, words) for a in sees])
    # bits past the sequence's rows are not looked at
    for b, (c, n) in enumerate(lens):
        for j in range(n, 32 * words):
            tree[g.start[b]:g.start[b + 1], j // 32] |= np.uint32(1 << (j % 32))
    q = rng.standard_normal((g.T, h, 576))
    out, lse = run_attend(m, g, q, 0.1, R.kind(fmt), tree=tree)
    check_attend(g, q, 0.1, out, lse, sees)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("ctx", [0, 40, 100])
def test_attend_masks_that_leave_rows_empty_and_nan_rows(m, cuda_lib, fmt, ctx):
    """Token 0 sees nothing of the draft (with ctx = 0: nothing at all); rows 1, 3 hold NaN and infinity: tokens
    that see one are NaN, the others are as if it were not there."""
    n = 6
    g = Paged(cuda_lib, [(ctx, n)], fmt, 512, 64, seed=4)
    fill(g, 4)
    at = g.rows(0, 0, ctx + n)
    sees = np.zeros((n, n), bool)
    for i in range(1, n):
        sees[i, i] = True
        sees[i, 2] = True
    rows = g.host[at].copy()
    if R.is_fp8(fmt):
        rows[ctx + 1, 512 + 128 + 3] = 255
        rows[ctx + 3, 512 + 128:512 + 128 + 16] = 255
    else:
        v = rows[ctx + 1].view(np.uint16)
        v[100] = 0x7FFF
        v = rows[ctx + 3].view(np.uint16)
        v[:512] = 0x7C00 if fmt == R.F16 else 0x7F80
    g.host[at] = rows
    g.upload()
    q = np.random.default_rng(8).standard_normal((n, 128, 576))
    out, lse = run_attend(m, g, q, 0.1, R.kind(fmt), tree=pack_tree(sees, 1))
    for i in (1, 3):
        assert np.all(np.isnan(out[i])), i
    keep = [i for i in range(n) if i not in (1, 3)]
    kv = R.unpack(g.host[at], 512, fmt)
    vis = np.concatenate([np.ones((n, ctx), bool), sees], 1)[keep]
    want, wl, A, S = R.attend(R.rounded(q, R.kind(fmt))[keep], kv, vis, 0.1, 512)
    tol, tl = R.attend_bounds(want, wl, A, S, R.kind(fmt))
    assert np.all(np.abs(out[keep] - want) <= tol)
    assert np.all((np.abs(lse[keep] - wl) <= tl) | (np.isneginf(wl) & np.isneginf(lse[keep])))
    if ctx == 0:
        assert np.all(out[0] == 0) and np.all(np.isneginf(lse[0]))


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("column", [5, 300, 540])
def test_attend_one_nan_spoils_the_whole_row_that_sees_it(m, cuda_lib, fmt, column):
    """A NaN in one half of a drafted row's latent values, or in its rotary ones, reaches every output of the tokens
    that see it, in both halves, call after call; the others are as without it."""
    lens = [(3 + 70 * k, 4) for k in range(40)]
    g = Paged(cuda_lib, lens, fmt, 512, 64, seed=5)
    fill(g, 5)
    sees = np.tril(np.ones((4, 4), bool))
    sees[3, 2] = False
    for b, (c, n) in enumerate(lens):
        row = g.host[g.rows(b, c + 2, c + 3)].copy()
        if R.is_fp8(fmt) and column < 512:
            row[0, 640 + column // 32] = 255
        else:
            at = column if not R.is_fp8(fmt) else 256 + column - 512
            row.view(np.uint16)[0, at] = 0x7FFF
        g.host[g.rows(b, c + 2, c + 3)] = row
    g.upload()
    q = np.random.default_rng(4).standard_normal((g.T, 16, 576))
    tree = np.tile(pack_tree(sees, 1), (len(lens), 1))
    t = R.kind(fmt)
    for _ in range(5):
        out, lse = run_attend(m, g, q, 0.1, t, tree=tree)
        for b, (c, n) in enumerate(lens):
            o = out[g.start[b]:g.start[b + 1]]
            assert np.all(np.isnan(o[2])) and not np.any(np.isnan(o[[0, 1, 3]])), b
    keep = [0, 1, 3]
    for b in (0, 1, 39):
        c, n = lens[b]
        kv = R.unpack(g.host[g.rows(b, 0, c + n)], 512, fmt)
        vis = np.concatenate([np.ones((n, c), bool), sees], 1)[keep]
        sl = slice(g.start[b], g.start[b + 1])
        want, wl, A, S = R.attend(R.rounded(q[sl], t)[keep], kv, vis, 0.1, 512)
        tol, tl = R.attend_bounds(want, wl, A, S, t)
        assert np.all(np.abs(out[sl][keep] - want) <= tol) and np.all(np.abs(lse[sl][keep] - wl) <= tl)


def test_bounds_out_of_range_skip_the_sequence(m, cuda_lib):
    """A sequence whose rows pass the call's, or whose context is negative, is skipped by the attention; one whose
    context passes its page table sees what the table holds; both are reported, the others are right."""
    F = cuda_lib
    lens = [(40, 2), (70, 3), (9, 2)]
    g = Paged(F, lens, R.FP8_BF16, 256, 16, seed=2)
    fill(g, 2)
    q = np.random.default_rng(3).standard_normal((7, 20, 320))
    chain = [np.tril(np.ones((n, n), bool)) for _, n in lens]
    for starts, ctx in (([0, 2, 5, 9], [40, 70, 9]), ([0, 2, 5, 7], [40, 70, -1])):
        g.bufs[0], g.bufs[1] = dev(np.array(starts, np.int32)), dev(np.array(ctx, np.int32))
        out, lse = run_attend(m, g, q, 0.2, "bf16", check=False)
        with pytest.raises(F.MoeError, match="bounds"):
            m.check_error()
        two = [(40, 2), (70, 3)]
        g.lens, keep = two, g.lens
        check_attend(g, q, 0.2, out, lse, chain[:2])
        g.lens = keep
        assert np.all(out[5:] == 7) and np.all(lse[5:] == 7)
    # a context past the table (5 pages of 16 rows): the 80 rows that the table holds, of which 73 to 79 were never
    # written and hold NaN patterns, so every weighted sum over them is NaN
    g.bufs[0], g.bufs[1] = dev(g.start), dev(np.array([40, 10 ** 6, 9], np.int32))
    out, lse = run_attend(m, g, q, 0.2, "bf16", check=False)
    with pytest.raises(F.MoeError, match="bounds"):
        m.check_error()
    assert np.all(np.isnan(out[2:5])) and np.all(np.isfinite(out[5:]))
    g.lens = [(40, 2)]
    check_attend(g, q, 0.2, out, lse, chain[:1])


@pytest.mark.parametrize("fmt", [R.F16, R.FP8_BF16])
def test_attend_strides(m, cuda_lib, fmt):
    """Padded rows; heads in front of tokens; no lse."""
    lens = [(77, 3), (10, 2)]
    g = Paged(cuda_lib, lens, fmt, 256, 32, seed=6)
    fill(g, 6)
    q = np.random.default_rng(6).standard_normal((g.T, 20, 320))
    chain = [np.tril(np.ones((n, n), bool)) for _, n in lens]
    for pad, hm in ((1, False), (0, True), (2, True)):
        out, lse = run_attend(m, g, q, 0.15, R.kind(fmt), pad=pad, head_major=hm, lse=pad != 1)
        check_attend(g, q, 0.15, out, lse, chain)


def test_attend_rows_outside_the_sequences_stay(m, cuda_lib):
    """Rows in front of the first sequence and behind the last are left as they were."""
    lens = [(30, 2), (9, 3)]
    g = Paged(cuda_lib, lens, R.BF16, 128, 16, q0=2)
    fill(g)
    q = np.random.default_rng(1).standard_normal((9, 4, 192))
    out, lse = run_attend(m, g, q, 0.2, "bf16", batch=g.batch(9))
    check_attend(g, q, 0.2, out, lse, [np.tril(np.ones((n, n), bool)) for _, n in lens])
    assert np.all(out[:2] == 7) and np.all(out[7:] == 7) and np.all(lse[:2] == 7) and np.all(lse[7:] == 7)


@pytest.mark.parametrize("fmt", [R.F16, R.BF16, R.FP8_BF16])
def test_attend_growing_scores(m, cuda_lib, fmt):
    """The running maximum moves in most tiles, upwards by far more than a step, and in others stays behind."""
    n_rows = 1500
    g = Paged(cuda_lib, [(n_rows - 1, 1)], fmt, 512, 64)
    rng = np.random.default_rng(0)
    k = rng.standard_normal((n_rows, 576)).astype(np.float32) * 0.2
    k[:, 0] = np.linspace(-60, 60, n_rows)
    k[::97, 0] = 75
    k[:, 32:64] = 0
    g.host[g.rows(0, 0, n_rows)] = R.pack(k[:, :512], k[:, 512:], fmt)
    g.upload()
    q = rng.standard_normal((1, 128, 576)) * 0.2
    q[0, :, 0] = np.linspace(-3, 3, 128)
    out, lse = run_attend(m, g, q, 1.0, R.kind(fmt))
    check_attend(g, q, 1.0, out, lse, [np.ones((1, 1), bool)])


def test_attend_large_negative_and_zero_scale(m, cuda_lib):
    g = Paged(cuda_lib, [(500, 2)], R.BF16, 512, 64)
    fill(g)
    q = np.random.default_rng(2).standard_normal((2, 128, 576))
    for scale in (0.0, -0.1, 3.0):
        out, lse = run_attend(m, g, q, scale, "bf16")
        check_attend(g, q, scale, out, lse, [np.tril(np.ones((2, 2), bool))])


def test_attend_same_bits_each_time(m, cuda_lib):
    """Partial results are joined in a fixed order: two calls give the same bits."""
    g = Paged(cuda_lib, [(9000, 3), (100, 1)], R.FP8_BF16, 512, 64)
    fill(g)
    q = np.random.default_rng(2).standard_normal((4, 128, 576))
    a, la = run_attend(m, g, q, 0.1, "bf16")
    b, lb = run_attend(m, g, q, 0.1, "bf16")
    assert np.array_equal(a, b) and np.array_equal(la, lb)


def test_offsets_past_32_bits(m, cuda_lib):
    """Pages whose byte offset passes 2^32 (a 5.9 GB cache, only the used pages written)."""
    import torch
    F = cuda_lib
    page, latent, fmt = 64, 512, R.BF16
    n_pages = 80000
    store = torch.empty(n_pages * page * 1152, dtype=torch.uint8, device="cuda")
    kv = F.KVCache(store, fmt, latent, page, n_pages)
    table = np.array([[n_pages - 1, 58255, 3, n_pages - 2]], np.int32)   # 58255 * 64 * 1152 is just below 2^32
    start, ctx = np.array([0, 200], np.int32), np.array([0], np.int32)
    bufs = [dev(start), dev(ctx), dev(table)]
    rng = np.random.default_rng(3)
    raw, x = typed(rng.standard_normal((200, 576)), "bf16")
    d = dev(raw)
    y = torch.zeros((200, 576), dtype=torch.int16, device="cuda")
    ready(m)
    m.kv_write_device(kv, F.KVBatch(1, 200, *bufs, 4), d, 30, 576)
    m.kv_read_device(kv, F.KVBatch(1, 200, *bufs, 4), y, 30, 576)
    m.check_error()
    assert np.array_equal(back(y, "bf16"), x)

    class G:
        pass
    g = G()
    g.kv, g.lens, g.start, g.fmt, g.latent = kv, [(199, 1)], np.array([0, 1]), fmt, latent
    b2 = [dev(np.array([0, 1], np.int32)), dev(np.array([199], np.int32)), bufs[2]]
    q = rng.standard_normal((1, 128, 576))
    out, lse = run_attend(m, g, q, 0.1, "bf16", batch=F.KVBatch(1, 1, *b2, 4))
    want, wl, A, S = R.attend(R.rounded(q, "bf16"), x, np.ones((1, 200), bool), 0.1, 512)
    tol, tl = R.attend_bounds(want, wl, A, S, "bf16")
    assert np.all(np.abs(out - want) <= tol) and np.all(np.abs(lse - wl) <= tl)
    del store


def test_graph_replay_and_two_streams(m, cuda_lib):
    """write -> attend captured once and replayed with new inputs and lengths; two graphs on two streams with their
    own workspaces replayed at once."""
    import torch
    F = cuda_lib
    sets = []
    for k in range(2):
        g = Paged(F, [(400 + 100 * k, 2), (90, 1)], R.FP8_BF16, 512, 64, seed=k)
        fill(g, k)
        s = torch.cuda.Stream()
        T, h = g.T, 128
        e = dict(g=g, s=s, kv=torch.zeros(T, 576, device="cuda"), ql=torch.zeros(T, h, 512, dtype=torch.bfloat16, device="cuda"),
                 qr=torch.zeros(T, h, 64, dtype=torch.bfloat16, device="cuda"), out=torch.zeros(T, h, 512, dtype=torch.bfloat16, device="cuda"),
                 lse=torch.zeros(T, h, device="cuda"), pos=dev(np.arange(T, dtype=np.int32)),
                 ws=torch.empty(m.mla_workspace_bytes(512), dtype=torch.uint8, device="cuda"))

        def step(e=e, g=g, s=s, h=h):
            m.kv_write_device(g.kv, g.batch(), e["kv"], 0, 576, None, 1e-6, F.RopeConfig(), e["pos"], s.cuda_stream)
            m.mla_attention_device(g.kv, g.batch(), e["ql"], (h * 512, 512), e["qr"], (h * 64, 64), h, 0.1, e["out"],
                                   (h * 512, 512), e["ws"], e["ws"].numel(), lse=e["lse"], stream=s.cuda_stream)
        torch.cuda.synchronize()
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        e["graph"] = graph
        sets.append(e)
    for rnd in range(3):
        for k, e in enumerate(sets):
            g, rng = e["g"], np.random.default_rng(10 * rnd + k)
            e["x"] = rng.standard_normal((g.T, 576)).astype(np.float32)
            e["q"] = rng.standard_normal((g.T, 128, 576))
            e["kv"].copy_(torch.from_numpy(e["x"]))
            e["ql"].copy_(torch.from_numpy(e["q"][..., :512]))
            e["qr"].copy_(torch.from_numpy(e["q"][..., 512:]))
            g.ctx = np.array([400 + 100 * k - 37 * rnd, 90 - rnd], np.int32)   # shorter contexts: rows behind them are stale
            g.bufs[1].copy_(torch.from_numpy(g.ctx))
            g.lens = [(int(c), n) for c, (_, n) in zip(g.ctx, g.lens)]
        torch.cuda.synchronize()
        for e in sets:
            with torch.cuda.stream(e["s"]):
                e["graph"].replay()
        torch.cuda.synchronize()
        m.check_error()
        for e in sets:
            g = e["g"]
            g.host = g.d.cpu().numpy()
            for b, (c, n) in enumerate(g.lens):   # the appended rows are this round's
                sl = slice(g.start[b], g.start[b + 1])
                rot = R.rotate(e["x"][sl, 512:].astype(np.float64), np.arange(g.start[b], g.start[b + 1]), R.freqs())
                want = R.pack(e["x"][sl, :512], rot, g.fmt)
                assert np.array_equal(g.host[g.rows(b, c, c + n)][:, :512], want[:, :512])
            check_attend(g, e["q"], 0.1, e["out"].float().cpu().numpy().astype(np.float64), e["lse"].cpu().numpy().astype(np.float64),
                         [np.tril(np.ones((n, n), bool)) for _, n in g.lens])
    for e in sets:
        del e["graph"]


def test_decode_steps_match_the_oracle(m, cuda_lib, oracle):
    """The operators as a decode step uses them (projections in numpy, rotary positions, append, attention here),
    against the oracle's mla_forward over several positions of a growing fp16 cache."""
    import torch
    F = cuda_lib
    cfg = oracle.mla_cfg(H=512, n_heads=8)
    from test_mla_oracle import _weights
    rng = np.random.default_rng(7)
    w = _weights(cfg, rng)
    H16 = lambda a: a.view(np.float16).astype(np.float64)   # noqa: E731
    g = Paged(F, [(0, 1)], R.F16, 512, 16, extra=2)
    g.table = np.zeros((1, 2), np.int32)
    g.table[0] = [2, 0]
    g.bufs[2], g.per = dev(g.table), 2
    rope = F.RopeConfig()
    ms = 0.1 * np.log(40.0) + 1.0
    scale = float(ms * ms / np.sqrt(cfg.qk_nope + cfg.qk_rope))
    cache = oracle.MlaCache(cfg, 32)
    QK = cfg.qk_nope + cfg.qk_rope
    for step in range(20):
        h = rng.standard_normal(cfg.H).astype(np.float32)
        want = oracle.mla_decode(cfg, w, h, cache, step)
        x = h.astype(np.float64)
        normed = R.rmsnorm(x, w["attn_norm"], float(cfg.eps))
        qf = (H16(w["q_b"]) @ R.rmsnorm(H16(w["q_a"]) @ normed, w["q_a_norm"], float(cfg.eps))).reshape(cfg.n_heads, QK)
        kva = (H16(w["kv_a"]) @ normed).astype(np.float32)
        qabs = np.einsum("hrd,hd->hr", H16(w["k_b"]), qf[:, :cfg.qk_nope])
        # rotary positions of the query heads on the device, in fp32
        pe, pos = dev(qf[:, cfg.qk_nope:].astype(np.float32)), dev(np.array([step], np.int32))
        pr = torch.zeros_like(pe)
        g.bufs[1] = dev(np.array([step], np.int32))
        ready(m)
        m.rope_device(rope, pe, 0, (8 * 64, 64), pr, 0, (8 * 64, 64), pos, 1, 8, 64)
        m.kv_write_device(g.kv, g.batch(), dev(kva), 0, 576, dev(w["kv_a_norm"]), float(cfg.eps), rope, pos)
        m.check_error()
        q = np.concatenate([qabs, pr.cpu().numpy().astype(np.float64)], -1)[None]
        out, _ = run_attend(m, g, q, scale, "f16")
        att = np.einsum("hvr,hr->hv", H16(w["v_b"]), out[0]).reshape(-1)
        got = x + H16(w["o_proj"]) @ att
        # fp16 queries, rows, weights and result: four roundings of 2^-11, on a sum that may cancel
        delta = np.abs(H16(w["o_proj"])) @ np.abs(att)
        assert np.max(np.abs(got - want) / delta) < 8 * 2.0 ** -11, step
        # the appended row is the oracle's, rounded to fp16
        row = R.unpack(g.d.cpu().numpy()[g.rows(0, step, step + 1)], 512, R.F16)[0]
        ref = np.concatenate([cache.c_kv[step], cache.k_rope[step]])
        assert np.max(np.abs(row - ref)) <= 2 * 2.0 ** -11 * np.max(np.abs(ref))


def test_entry_points_refuse(m, cuda_lib):
    """What the host checks refuse comes back as an error with a message, and launches nothing."""
    import torch
    F = cuda_lib
    g = Paged(F, [(8, 1)], R.BF16, 128, 8)
    ws = torch.empty(m.mla_workspace_bytes(128), dtype=torch.uint8, device="cuda")
    x = torch.zeros(8, 192, device="cuda")
    before = m.kernel_launches
    with pytest.raises(F.MoeError, match="page_size"):
        m.kv_write_device(F.KVCache(g.d, R.BF16, 128, 12, g.n_pages), g.batch(), x, 0, 192)
    with pytest.raises(F.MoeError, match="format"):
        m.kv_read_device(F.KVCache(g.d, 5, 128, 8, g.n_pages), g.batch(), x, 0, 192)
    with pytest.raises(F.MoeError, match="overlap"):
        m.kv_read_device(g.kv, g.batch(2), x, 0, 191)
    with pytest.raises(F.MoeError, match="workspace"):
        m.mla_attention_device(g.kv, g.batch(), x, (128, 128), x, (64, 64), 1, 0.1, x, (128, 128), ws, ws.numel() - 1)
    with pytest.raises(F.MoeError, match="multiple of 8"):
        m.mla_attention_device(g.kv, g.batch(), x, (128, 129), x, (64, 64), 1, 0.1, x, (128, 128), ws, ws.numel())
    with pytest.raises(F.MoeError, match="even"):
        m.rope_device(F.RopeConfig(dim=7), x, 0, (192, 192), x, 0, (192, 192), g.bufs[1], 1, 1, 192)
    assert m.kernel_launches == before
    # nothing to do is no error
    m.kv_write_device(g.kv, F.KVBatch(0, 0, None, None, None, 0), None, 0, 192)
    m.mla_attention_device(g.kv, F.KVBatch(0, 4, None, None, None, 0), x, (128, 128), x, (64, 64), 1, 0.1, x, (128, 128), ws,
                           ws.numel())
    assert m.kernel_launches == before
    m.check_error()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("half", [False, True])
def test_rope_in_place_is_the_copy(m, cuda_lib, t, half):
    """Aligned rows in place: the rotated values have the bits of the out-of-place call, the others stay."""
    import torch
    T, H, D, off, dim = 9, 6, 192, 128, 64
    raw, _ = typed(np.random.default_rng(2).standard_normal((T, H, D)), t)
    d, y, p = dev(raw), torch.zeros_like(dev(raw)), dev(np.arange(T, dtype=np.int32) * 1001)
    cfg = cuda_lib.RopeConfig(dim=dim, half_layout=half)
    ready(m)
    m.rope_device(cfg, d, DT[t], (H * D, D), y, DT[t], (H * D, D), p, T, H, D, off)
    m.rope_device(cfg, d, DT[t], (H * D, D), d, DT[t], (H * D, D), p, T, H, D, off)
    m.check_error()
    assert np.array_equal(d.cpu().numpy(), y.cpu().numpy())
    assert np.array_equal(d.cpu().numpy()[..., :off], raw[..., :off]) and not np.array_equal(d.cpu().numpy(), raw)
