"""The operators of a language-model student on the GPU -- embedding, the gated pair of Linear layers, the distillation
loss -- against their formulas in 64 bits, at the sizes, views and masks where they can go wrong.

Tolerances count roundings: u is half a step of the type (2^-24, 2^-53)."""
import ctypes as C
import fnmatch
import re
import zlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]
U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
ACTS = ["silu", "gelu", "relu", "sigmoid"]


def rng_of(*key):
    return np.random.default_rng([zlib.crc32(k.encode()) if isinstance(k, str) else int(k) for k in key])


def framed(tt, shape, dtype, margin=37):
    """A result tensor inside a larger buffer of a known pattern, and a check that the pattern around it is intact."""
    n = int(np.prod(shape))
    host = np.full(n + 2 * margin, 77.0, dtype)
    whole = tt.Tensor.from_numpy(host)
    t = tt.Tensor(whole.storage, whole.dtype, shape, None, margin)

    def intact():
        back = whole.to_numpy()
        return np.all(back[:margin] == 77.0) and np.all(back[margin + n:] == 77.0)

    return t, intact


# ---- embedding -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", [np.int32, np.int64, np.uint8, np.int16])
@pytest.mark.parametrize("shape, vocab, dim", [((1,), 1, 1), ((3,), 5, 1), ((2, 7), 11, 3), ((65,), 100, 4), ((1,), 100, 1024),
                                               ((5, 3), 40, 333), ((300,), 17, 66), ((9,), 120, 2051), ((0,), 7, 5)])
def test_embedding_rows(tt, dtype, index, shape, vocab, dim):
    r = rng_of(vocab, dim, 1)
    table = r.normal(0, 1, (vocab, dim)).astype(dtype)
    ids = r.integers(0, vocab, shape).astype(index)
    scale = 3.3
    out, intact = framed(tt, shape + (dim,), dtype)
    got = tt.embedding(tt.Tensor.from_numpy(ids), tt.Tensor.from_numpy(table), scale=scale, out=out)
    assert got is out
    assert np.array_equal(out.to_numpy(), table[ids.astype(np.int64)] * dtype(scale))  # one product, rounded once: exact
    assert intact()


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_views_and_padding(tt, dtype):
    r = rng_of(3)
    base = r.normal(0, 1, (64, 50)).astype(dtype)
    ids = np.array([[0, 49, 7], [-1, 50, 3]], np.int64)
    t = tt.Tensor.from_numpy(base)
    tied = t.permute(1, 0)  # a Linear weight [in, out] as a table of `out` rows, read in place
    got = tt.embedding(tt.Tensor.from_numpy(ids), tied, scale=0.5).to_numpy()
    want = np.where(((ids >= 0) & (ids < 50))[..., None], base.T[np.clip(ids, 0, 49)] * dtype(0.5), dtype(0))
    assert np.array_equal(got, want)
    # rows further apart than they are long, a first element off every boundary
    part = tt.Tensor(t.storage, t.dtype, (40, 31), (50, 1), 53)
    ids2 = r.integers(-3, 43, (70,)).astype(np.int32)
    rows = base.reshape(-1)[53:][np.arange(40)[:, None] * 50 + np.arange(31)]
    want = np.where(((ids2 >= 0) & (ids2 < 40))[:, None], rows[np.clip(ids2, 0, 39)], dtype(0))
    assert np.array_equal(tt.embedding(tt.Tensor.from_numpy(ids2), part).to_numpy(), want)
    # one row for every token, and indices that are a strided view themselves
    one = tt.Tensor(t.storage, t.dtype, (9, 50), (0, 1), 100)
    idv = tt.Tensor.from_numpy(np.arange(12, dtype=np.int32).reshape(3, 4)).permute(1, 0)
    got = tt.embedding(idv, one).to_numpy()
    assert got.shape == (4, 3, 50)
    want = np.where((np.arange(12).reshape(3, 4).T < 9)[..., None], base[2], dtype(0))
    assert np.array_equal(got, want)


def embedding_gradient(dy, ids, vocab, scale):
    """(gradient, sum of magnitudes, rows a token) in 64 bits."""
    g, m, n = np.zeros((vocab, dy.shape[-1])), np.zeros((vocab, dy.shape[-1])), np.zeros(vocab)
    ok = (ids >= 0) & (ids < vocab)
    np.add.at(g, ids[ok], dy[ok].astype(np.float64))
    np.add.at(m, ids[ok], np.abs(dy[ok]).astype(np.float64))
    np.add.at(n, ids[ok], 1)
    return g * scale, m * abs(scale), n


def check_embedding_gradient(got, dy, ids, vocab, scale, dtype, before=None):
    want, mag, n = embedding_gradient(dy, ids, vocab, scale)
    if before is not None:
        want = want + before
    # sums in 64 bits (n + 2 roundings of 2^-53 of the magnitudes, and the comparison's own sum as many), rounded once
    tol = U[dtype] * np.abs(want) + 2 * (n[:, None] + 3) * 2.0 ** -53 * (mag + (0 if before is None else np.abs(before)))
    assert np.all(np.abs(got.astype(np.float64) - want) <= tol)
    return n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", [np.int32, np.int64])
@pytest.mark.parametrize("count, vocab, dim", [(1, 1, 1), (1, 300, 8), (5, 3, 7), (16, 1, 4), (17, 1, 5), (257, 2, 3), (100, 1000, 333), (1000, 37, 130), (64, 9, 30), (65, 40, 1), (128, 3, 257), (128, 70000, 8), (129, 50, 12),
                                               (4096, 600, 64), (3000, 140000, 12), (700, 513, 1028), (0, 9, 6), (5000, 1, 260)])
def test_embedding_gradient(tt, dtype, index, count, vocab, dim):
    r = rng_of(count, vocab, dim)
    dy = r.normal(0, 1, (count, dim)).astype(dtype)
    ids = (r.random(count) ** 3 * (vocab + 2)).astype(index) - 1  # a few tokens often; -1 and vocab: padding
    out, intact = framed(tt, (vocab, dim), dtype)
    tt.embedding_backward(tt.Tensor.from_numpy(dy), tt.Tensor.from_numpy(ids), vocab, scale=1.7, out=out)
    got = out.to_numpy()
    n = check_embedding_gradient(got, dy, ids, vocab, 1.7, dtype)
    assert np.all(got[n == 0] == 0)
    assert intact()
    # the same bits again, and added to what is there
    again = tt.embedding_backward(tt.Tensor.from_numpy(dy), tt.Tensor.from_numpy(ids), vocab, scale=1.7).to_numpy()
    assert np.array_equal(got, again)
    before = r.normal(0, 1, (vocab, dim)).astype(dtype)
    acc = tt.Tensor.from_numpy(before)
    tt.embedding_backward(tt.Tensor.from_numpy(dy), tt.Tensor.from_numpy(ids), vocab, scale=1.7, out=acc, accumulate=True)
    check_embedding_gradient(acc.to_numpy(), dy, ids, vocab, 1.7, dtype, before.astype(np.float64))
    assert np.array_equal(acc.to_numpy()[n == 0], before[n == 0])


@pytest.mark.parametrize("vocab", [130560, 130561, 130817, 131071, 131072, 131073, 262144])
@pytest.mark.parametrize("index", [np.int32, np.int64])
def test_embedding_gradient_fullest_buckets(tt, vocab, index):
    """Vocabularies whose buckets hold as many tokens as the counters have room for, or one fewer or more; first and last token."""
    count, dim = 6000, 5
    r = rng_of(vocab, 17)
    ids = r.integers(0, vocab, count)
    ids[:700] = 256 * r.integers(0, vocab // 256, 700) + 3  # more positions of one bucket than a wave lists
    ids[700:710], ids[710:720], ids[720:725], ids[725:730] = 0, vocab - 1, -1, vocab
    ids = ids.astype(index)
    dy = r.integers(-8, 9, (count, dim)).astype(np.float32)  # whole numbers: the sums are exact
    out, intact = framed(tt, (vocab, dim), np.float32)
    tt.embedding_backward(tt.Tensor.from_numpy(dy), tt.Tensor.from_numpy(ids), vocab, out=out)
    assert np.array_equal(out.to_numpy().astype(np.float64), embedding_gradient(dy, ids, vocab, 1.0)[0])
    assert intact()


@pytest.mark.parametrize("pattern", ["one", "blocks", "bucket", "borders"])
def test_embedding_gradient_runs(tt, pattern):
    """Runs of equal tokens that fill, end at, cross and span the groups that are added up together."""
    count, vocab, dim = 2048, 1024, 20
    i = np.arange(count)
    ids = {"one": np.full(count, 5), "blocks": i // 16, "bucket": (i * 7 % 4) * 256 + 3, "borders": np.where(i < 15, 1, np.where(i < 33, 2, np.where(i < 48, 3, 4 + i // 100)))}[pattern]
    r = rng_of(7)
    ids = ids[r.permutation(count)].astype(np.int32)
    dy = r.integers(-8, 9, (count, dim)).astype(np.float32)  # whole numbers: the sums are exact
    got = tt.embedding_backward(tt.Tensor.from_numpy(dy), tt.Tensor.from_numpy(ids), vocab).to_numpy()
    assert np.array_equal(got.astype(np.float64), embedding_gradient(dy, ids, vocab, 1.0)[0])


@pytest.mark.parametrize("dtype, count, vocab, dim", [(np.float32, 70000, 300, 520), (np.float32, 4097, 5, 2047), (np.float64, 40000, 30000, 421), (np.float32, 30000, 3, 64)])
def test_embedding_gradient_of_many(tt, dtype, count, vocab, dim):
    """Long lists: chunks of both lengths, tokens of thousands of positions, rows loaded past the caches; the forward too."""
    r = rng_of(count, vocab, dim)
    ids = ((vocab + 1) ** r.random(count) - 1).astype(np.int64)
    dy = r.integers(-8, 9, (64, dim)).astype(dtype)[r.integers(0, 64, count)]  # whole numbers: the sums are exact
    got = tt.embedding_backward(tt.Tensor.from_numpy(dy), tt.Tensor.from_numpy(ids), vocab).to_numpy()
    want = np.zeros((vocab, dim))
    order = np.argsort(ids, kind="stable")
    starts = np.flatnonzero(np.r_[True, np.diff(ids[order]) > 0])
    want[ids[order][starts]] = np.add.reduceat(dy[order].astype(np.float64), starts, axis=0)
    assert np.array_equal(got.astype(np.float64), want)
    table = r.integers(-100, 101, (vocab, dim)).astype(dtype)
    assert np.array_equal(tt.embedding(tt.Tensor.from_numpy(ids), tt.Tensor.from_numpy(table), scale=0.5).to_numpy(), table[ids] * dtype(0.5))


# ---- the gated pair ------------------------------------------------------------------------------------------------------


def erf(x):
    from scipy.special import erf as f
    return f(x)


def act_of(g, act):
    if act == "relu":
        return np.maximum(g, 0), np.where(g < 0, 0.0, 1.0)
    if act == "gelu":
        cdf = 0.5 * (1 + erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * np.exp(-0.5 * g * g) / (2 * np.pi) ** 0.5
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-g))
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def act_error(g, act, u):
    """Bounds of |act(g)|'s and |act'(g)|'s errors.  s = 1 / (1 + exp(-g)): exp within 2 steps (4 u), a sum, a quotient: 6 u
    of s, and 7 u absolute in 1 - s; the products add a few u each.  erf within 2 steps of a value up to 1 (4 u), its
    argument's rounding 1 u more, halved: 3 u absolute in the distribution function, 8 u with the products."""
    if act == "relu":
        return 0 * g, 0 * g
    value = 8 * u * (np.ones_like(g) if act == "sigmoid" else np.abs(g))
    return value, 20 * u * (1 + np.abs(g))


def gated_reference(x, wg, wu, bg, bu, act):
    x, wg, wu = (a.astype(np.float64) for a in (x, wg, wu))
    g, u = x @ wg, x @ wu
    if bg is not None:
        g = g + bg.astype(np.float64)
    if bu is not None:
        u = u + bu.astype(np.float64)
    return g, u


def product_error(a, b, u, extra=0.0):
    """(terms + 2) roundings of the magnitudes: an inner product of any order of summation, and a bias."""
    return (a.shape[1] + 2 + extra) * u * (np.abs(a).astype(np.float64) @ np.abs(b).astype(np.float64))


def check_gated(tt, dtype, act, x, wg, wu, bg, bu, tx, twg, twu, dh=None, save=True):
    u_ = U[dtype]
    put = lambda a: tt.Tensor.from_numpy(a) if a is not None else None  # noqa: E731
    hidden = wg.shape[1]
    g, u = gated_reference(x, wg, wu, bg, bu, act)
    eg = product_error(x, wg, u_) + (u_ * np.abs(bg) if bg is not None else 0)
    eu = product_error(x, wu, u_) + (u_ * np.abs(bu) if bu is not None else 0)
    value, slope = act_of(g, act)
    ev, _ = act_error(g, act, u_)
    th = framed(tt, (x.shape[0], hidden), dtype)
    plain = tt.gated_linear(tx, twg, twu, put(bg), put(bu), activation=act, out=th[0])
    assert plain is th[0] and th[1]()
    h, sg, su = tt.gated_linear(tx, twg, twu, put(bg), put(bu), activation=act, save=True)
    # act' is at most 1.13 in magnitude for these, so an error of g reaches act(g) 1.2 times at most
    tol = (ev + 1.2 * eg) * (np.abs(u) + eu) + np.abs(value) * eu + 2 * u_ * np.abs(value * u)
    for got in (plain.to_numpy(), h.to_numpy()):
        assert np.all(np.abs(got - value * u) <= tol + 1e-300)
    assert np.all(np.abs(sg.to_numpy() - g) <= eg) and np.all(np.abs(su.to_numpy() - u) <= eu)
    if dh is None:
        return
    # backward from the saved g and u as they are
    g, u = sg.to_numpy().astype(np.float64), su.to_numpy().astype(np.float64)
    value, slope = act_of(g, act)
    ev, es = act_error(g, act, u_)
    d = dh.astype(np.float64)
    dg, du = d * u * slope, d * value
    edg, edu = np.abs(d * u) * es + 3 * u_ * np.abs(dg), np.abs(d) * ev + 2 * u_ * np.abs(du)
    want = (dg @ wg.T.astype(np.float64) + du @ wu.T.astype(np.float64), x.T.astype(np.float64) @ dg, x.T.astype(np.float64) @ du,
            dg.sum(0), du.sum(0))
    tol = (edg @ np.abs(wg.T) + edu @ np.abs(wu.T) + product_error(np.concatenate([dg, du], 1), np.concatenate([wg.T, wu.T], 0), u_, 2),
           np.abs(x.T) @ edg + product_error(x.T, dg, u_), np.abs(x.T) @ edu + product_error(x.T, du, u_),
           edg.sum(0) + (len(dg) + 2) * u_ * np.abs(dg).sum(0), edu.sum(0) + (len(du) + 2) * u_ * np.abs(du).sum(0))
    frames = [framed(tt, w.shape, dtype) for w in want]
    got = tt.gated_linear_backward(put(dh), tx, twg, twu, sg, su, activation=act, out=tuple(f[0] for f in frames))
    for name, a, w, t, f in zip(("dx", "dwg", "dwu", "dbg", "dbu"), got, want, tol, frames):
        assert np.all(np.abs(a.to_numpy() - w) <= t + 1e-300), name
        assert f[1](), name
    none = tt.gated_linear_backward(put(dh), tx, twg, twu, sg, su, activation=act, bias_grad=False)
    assert none[3] is None and none[4] is None
    for a, b in zip(got[:3], none[:3]):
        assert np.array_equal(a.to_numpy(), b.to_numpy())


def gated_data(r, dtype, rows, inner, hidden):
    n = lambda *s: r.normal(0, 1, s).astype(dtype)  # noqa: E731
    return n(rows, inner), (n(inner, hidden) * inner ** -0.5).astype(dtype), (n(inner, hidden) * inner ** -0.5).astype(dtype), n(hidden), n(hidden), n(rows, hidden)


SIZES = [(1, 1, 1), (1, 5, 3), (1, 64, 128), (2, 333, 70), (3, 1024, 260), (5, 48, 1000), (8, 200, 516), (9, 128, 256), (16, 96, 33), (17, 64, 64), (33, 100, 77),
         (64, 64, 128), (65, 40, 132), (130, 260, 192), (128, 256, 1024), (300, 17, 130), (257, 512, 384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows, inner, hidden", SIZES)
def test_gated_linear(tt, dtype, act, rows, inner, hidden):
    r = rng_of(rows, inner, hidden, act)
    x, wg, wu, bg, bu, dh = gated_data(r, dtype, rows, inner, hidden)
    both = (rows + hidden) % 3
    bg, bu = (bg, bu) if both == 0 else (bg, None) if both == 1 else (None, None)
    check_gated(tt, dtype, act, x, wg, wu, bg, bu, *(tt.Tensor.from_numpy(a) for a in (x, wg, wu)), dh=dh)


@pytest.mark.parametrize("rows, inner, hidden", [(1024, 784, 1024), (1024, 1024, 516), (2048, 512, 1536), (512, 2048, 256), (16, 1024, 4096), (130, 4096, 512)])
def test_gated_linear_large(tt, rows, inner, hidden):
    r = rng_of(rows, inner, hidden)
    x, wg, wu, bg, bu, dh = gated_data(r, np.float32, rows, inner, hidden)
    check_gated(tt, np.float32, "silu", x, wg, wu, bg, bu, *(tt.Tensor.from_numpy(a) for a in (x, wg, wu)), dh=dh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 4, 11, 70, 256])
@pytest.mark.parametrize("form", ["transposed", "packed", "padded", "offset", "strided", "tied", "expanded"])
def test_gated_linear_views(tt, dtype, rows, form):
    inner, hidden = 96, 160
    r = rng_of(rows, form)
    x, wg, wu, bg, bu, dh = gated_data(r, dtype, rows, inner, hidden)
    T = tt.Tensor
    tx, twg, twu = (T.from_numpy(a) for a in (x, wg, wu))
    if form == "transposed":
        tx, twg, twu = (T.from_numpy(np.ascontiguousarray(a.T)).permute(1, 0) for a in (x, wg, wu))
    elif form == "packed":    # gate and up side by side in one weight
        w = T.from_numpy(np.concatenate([wg, wu], 1))
        twg, twu = (T(w.storage, w.dtype, (inner, hidden), (2 * hidden, 1), o) for o in (0, hidden))
    elif form == "padded":
        def padded(a, extra):
            t = T.from_numpy(np.concatenate([a, np.full((a.shape[0], extra), np.nan, dtype)], 1))
            return T(t.storage, t.dtype, a.shape, (a.shape[1] + extra, 1), 0)
        tx, twg, twu = padded(x, 4), padded(wg, 3), padded(wu, 8)
    elif form == "offset":
        def moved(a):
            t = T.from_numpy(np.concatenate([np.full(3, np.nan, dtype), a.reshape(-1)]))
            return T(t.storage, t.dtype, a.shape, (a.shape[1], 1), 3)
        tx, twg, twu = moved(x), moved(wg), moved(wu)
    elif form == "strided":
        def spread(a):
            b = np.full((a.shape[0], a.shape[1], 2), np.nan, dtype)
            b[..., 0] = a
            t = T.from_numpy(b)
            return T(t.storage, t.dtype, a.shape, (2 * a.shape[1], 2), 0)
        tx, twg, twu = spread(x), spread(wg), spread(wu)
    elif form == "tied":      # one weight for both
        wu, twu = wg, twg
    else:                     # the same row for every position
        x = np.repeat(x[:1], rows, 0)
        tx = T(tx.storage, tx.dtype, (rows, inner), (0, 1), 0)
    check_gated(tt, dtype, "silu", x, wg, wu, bg, None, tx, twg, twu, dh=dh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, inner, hidden", [(n, *s) for s in ((1, 2), (7, 3), (16, 31), (17, 33), (250, 64), (1003, 130))
                                                 for n in (3, 5, 8, 15, 16, 17, 31, 33, 64, 100, 250)] + [(5, 300, 8200), (17, 300, 8200), (33, 300, 8200)])
def test_gated_linear_blocks_of_rows(tt, dtype, rows, inner, hidden):
    """Row counts, reductions and widths around the blocks of 16 and 32 rows, 8 or 16 k and 32 columns; operands are cut out of
    buffers of NaN, which nothing may reach."""
    T = tt.Tensor
    r = rng_of(rows, inner, hidden, "rows")
    x, wg, wu, bg, bu, _ = gated_data(r, dtype, rows, inner, hidden)

    def inside(a):
        b = np.full((a.shape[0] + 2, a.shape[1] + 3), np.nan, dtype)
        b[1:-1, 1:-2] = a
        t = T.from_numpy(b)
        return T(t.storage, t.dtype, a.shape, (b.shape[1], 1), b.shape[1] + 1)

    check_gated(tt, dtype, "gelu" if rows % 2 else "silu", x, wg, wu, bg if rows % 3 else None, bu, inside(x), inside(wg), inside(wu))


def test_gated_linear_beyond_32_bit_offsets(tt):
    """Matrices of more than 2^31 bytes, and rows that lie that far apart: whole numbers, so every sum is exact."""
    r = rng_of(31)
    T = tt.Tensor
    rows, inner, hidden = 300, 4, 1 << 20
    x, wg, wu = r.integers(-2, 3, (rows, inner)).astype(np.float64), *(r.integers(-2, 3, (inner, hidden)).astype(np.float64) for _ in range(2))
    dh = T.from_numpy(r.integers(-1, 2, (1, hidden)).astype(np.float64)).expand((rows, hidden))
    tx, twg, twu = (T.from_numpy(a) for a in (x, wg, wu))
    h, g, u = tt.gated_linear(tx, twg, twu, activation="relu", save=True)
    part = lambda t, c: T(t.storage, t.dtype, (rows, 1000), (hidden, 1), c).contiguous().to_numpy()  # noqa: E731
    for c in (0, 1 << 19, hidden - 1000):
        wantg, wantu = x @ wg[:, c:c + 1000], x @ wu[:, c:c + 1000]
        assert np.array_equal(part(g, c), wantg) and np.array_equal(part(u, c), wantu) and np.array_equal(part(h, c), np.maximum(wantg, 0) * wantu)
    del h
    dx, dwg, dwu, dbg, dbu = (t.to_numpy() for t in tt.gated_linear_backward(dh, tx, twg, twu, g, u, activation="relu"))
    d, sum_dx = T(dh.storage, dh.dtype, (hidden,), (1,), 0).to_numpy(), np.zeros((rows, inner))
    for c in range(0, hidden, 1 << 16):
        s = slice(c, c + (1 << 16))
        wantg, wantu = x @ wg[:, s], x @ wu[:, s]
        pg, pu = d[s] * wantu * (wantg >= 0), d[s] * np.maximum(wantg, 0)
        assert np.array_equal(dwg[:, s], x.T @ pg) and np.array_equal(dwu[:, s], x.T @ pu)
        assert np.array_equal(dbg[s], pg.sum(0)) and np.array_equal(dbu[s], pu.sum(0))
        sum_dx += pg @ wg[:, s].T + pu @ wu[:, s].T
    assert np.array_equal(dx, sum_dx)
    del g, u
    # two rows of x 2^31 bytes apart
    far = T.empty(((1 << 28) + 64,), tt._capi.F64)
    for i, at in enumerate((0, 1 << 28)):
        T(far.storage, far.dtype, (40,), (1,), at).assign(T.from_numpy(np.arange(40, dtype=np.float64) + 100 * i))
    xf = T(far.storage, far.dtype, (2, 40), (1 << 28, 1), 0)
    host = np.stack([np.arange(40.0), np.arange(40.0) + 100])
    w = r.integers(-2, 3, (40, 24)).astype(np.float64)
    h, g, u = tt.gated_linear(xf, T.from_numpy(w), T.from_numpy(w), activation="relu", save=True)
    assert np.array_equal(g.to_numpy(), host @ w) and np.array_equal(h.to_numpy(), np.maximum(host @ w, 0) * (host @ w))
    ones = T.from_numpy(np.ones((2, 24)))
    got = tt.gated_linear_backward(ones, xf, T.from_numpy(w), T.from_numpy(w), g, u, activation="relu")
    pg, pu = (host @ w) * ((host @ w) >= 0), np.maximum(host @ w, 0)
    assert np.array_equal(got[1].to_numpy(), host.T @ pg) and np.array_equal(got[2].to_numpy(), host.T @ pu)


def test_gated_linear_largest_grids(tt):
    """Sizes whose workgroups one launch cannot hold: the copy of 2^26 rows of 257 elements (an overlapping view: element (r, c) is
    base[r + c]), and 2^26 columns of doubles for one row.  Whole numbers, so every sum is exact."""
    T = tt.Tensor
    r = rng_of(53)
    rows, inner = 1 << 26, 257
    base = r.integers(-1, 2, rows + inner).astype(np.float32)
    x = T(T.from_numpy(base).storage, tt._capi.F32, (rows, inner), (1, 1), 0)
    wg, wu = (r.integers(-1, 2, (inner, 1)).astype(np.float32) for _ in range(2))
    try:
        got = tt.gated_linear(x, T.from_numpy(wg), T.from_numpy(wu), activation="relu").to_numpy()[:, 0]
        some = np.unique(np.concatenate([np.arange(0, rows, 40009), r.integers(0, rows, 3000), np.arange(64), rows - 1 - np.arange(64)]))
        part = base[some[:, None] + np.arange(inner)]
        assert np.array_equal(got[some], np.maximum(part @ wg, 0)[:, 0] * (part @ wu)[:, 0])
        del x, got
        hidden = 1 << 26
        w = r.integers(-3, 4, (2, hidden)).astype(np.float64)
        gate, up = (T.from_numpy(w[i:i + 1]) for i in range(2))
        got = tt.gated_linear(T.from_numpy(np.array([[3.0]])), gate, up, activation="relu").to_numpy()
        assert np.array_equal(got[0], np.maximum(3 * w[0], 0) * (3 * w[1]))
    finally:
        tt._capi.lib.ttamd_empty_cache(0)  # (70 GB of workspace)


def gated_variant(tt, tx, twg, twu, backward=False):
    """The kernels that a call of these operands runs, without the prefix and the type."""
    v = [t.view2() for t in (tx, twg, twu)]
    name = tt._capi.lib.ttamd_gated_linear_variant(tx.dtype, *tx.shape, twg.shape[1], *(C.byref(a) for a in v), int(backward)).decode()
    return re.sub(r"^gated(_backward)?_f(32|64)_", "", name)


FORWARD_TILES = [(np.float32, "64x128", 269, 71, 71), (np.float32, "64x128", 260, 40, 72), (np.float32, "64x128_halves", 280, 253, 101),
                 (np.float32, "64x128_halves", 1000, 784, 1012), (np.float32, "128x128", 5630, 71, 130), (np.float32, "128x128", 5748, 36, 132),
                 (np.float32, "256x128", 1539, 100, 4588), (np.float32, "256x128", 5085, 50, 1429), (np.float64, "64x64", 258, 35, 74),
                 (np.float64, "64x64", 265, 68, 68), (np.float64, "128x128", 333, 50, 4345), (np.float64, "128x128", 261, 36, 4964),
                 (np.float64, "256x128", 721, 36, 4828), (np.float64, "256x128", 1227, 67, 2921)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype, tile, rows, inner, hidden", FORWARD_TILES)
def test_gated_linear_forward_tiles(tt, dtype, tile, rows, inner, hidden, act):
    """Every tile of the forward grid, sizes that are no multiples of it, whole vectors and not.  Inputs of 12 bits (f64: 29) and
    weights of -1, 0, 1, all times powers of two: g and u are exact, and no type of fewer bits could hold what they are made of."""
    bits = 11 if dtype is np.float32 else 28
    T, u_ = tt.Tensor.from_numpy, U[dtype]
    r = rng_of(rows, inner, hidden, act, "tiles")
    x = (r.integers(-2 ** bits + 1, 2 ** bits, (rows, inner)) * 2.0 ** -bits).astype(dtype)
    wg, wu = ((r.integers(-1, 2, (inner, hidden)) * 0.25).astype(dtype) for _ in range(2))
    bg, bu = (r.integers(-9, 10, hidden).astype(dtype) * dtype(0.25) for _ in range(2))
    tx, twg, twu = T(x), T(wg), T(wu)
    assert gated_variant(tt, tx, twg, twu) == tile
    g, u = gated_reference(x, wg, wu, bg, bu, act)
    assert (np.abs(x).sum(1).max() * 0.25 + 2.25) * 2.0 ** (bits + 2) < 1 / u_  # (exact in the type, in any order)
    h, sg, su = tt.gated_linear(tx, twg, twu, T(bg), T(bu), activation=act, out=(frame := framed(tt, (rows, hidden), dtype))[0], save=True)
    assert np.array_equal(sg.to_numpy(), g) and np.array_equal(su.to_numpy(), u) and frame[1]()
    value, _ = act_of(g, act)
    # the activation's roundings and the product's; in f64 the reference's own as well
    own = 2 if dtype is np.float64 else 1
    assert np.all(np.abs(h.to_numpy() - value * u) <= own * (act_error(g, act, u_)[0] + 2 * u_ * np.abs(value)) * np.abs(u))
    plain = tt.gated_linear(tx, twg, twu, T(bg), T(bu), activation=act).to_numpy()
    assert np.array_equal(plain, h.to_numpy())


BACKWARD_TILES = [(np.float32, "64x64", 138, 40, 68), (np.float32, "64x64_w*", 437, 36, 68), (np.float32, "64x64_x1", 140, 36, 248),
                  (np.float32, "64x64_x1_w*", 434, 36, 116), (np.float32, "64x64_x2", 145, 34, 383), (np.float32, "64x64_x2_w*", 351, 36, 324),
                  (np.float32, "128x128", 1766, 1948, 932), (np.float32, "128x128", 2022, 1923, 783), (np.float32, "128x128_w*", 1353, 1092, 68),
                  (np.float32, "128x128_w*", 1492, 1126, 67), (np.float32, "128x128_x1", 797, 1884, 1184), (np.float32, "128x128_x1", 898, 1617, 1397),
                  (np.float32, "128x128_x1_w*", 4295, 348, 1504), (np.float32, "128x128_x1_w*", 4465, 330, 1465),
                  (np.float32, "128x128_x16", 335, 348, 4460), (np.float32, "128x128_x4", 199, 1483, 1706),
                  (np.float32, "128x128_x4_w*", 4640, 72, 3088), (np.float32, "128x128_x4_w*", 4814, 67, 3201), (np.float64, "64x64", 138, 34, 74),
                  (np.float64, "64x64_w*", 427, 36, 76), (np.float64, "64x64_x1", 151, 36, 224), (np.float64, "64x64_x1_w*", 438, 37, 118),
                  (np.float64, "64x64_x2", 148, 33, 327), (np.float64, "64x64_x2_w*", 330, 36, 344)]


@pytest.mark.parametrize("wide", ["operands", "products"])
@pytest.mark.parametrize("dtype, tile, rows, inner, hidden", BACKWARD_TILES)
def test_gated_linear_backward_tiles(tt, dtype, tile, rows, inner, hidden, wide):
    """Every tile of the backward grid with whole and cut reductions, sizes that are no multiples of it, whole vectors and not.
    Whole numbers under relu, of 12 bits (f64: 29) on one side of each product and -1, 0, 1 on the other: every sum is exact, and
    no type of fewer bits could hold its terms."""
    T = tt.Tensor.from_numpy
    r = rng_of(rows, inner, hidden, wide)
    most = 4095 if dtype is np.float32 else 2 ** 29 - 1
    one = lambda *n: r.integers(-1, 2, n).astype(dtype)  # noqa: E731
    many = lambda *n: r.integers(-most, most + 1, n).astype(dtype)  # noqa: E731
    x, wg, wu = (many if wide == "operands" else one)(rows, inner), *((many if wide == "operands" else one)(inner, hidden) for _ in range(2))
    g, u = ((one if wide == "operands" else many)(rows, hidden) for _ in range(2))
    dh = one(rows, hidden)
    tx, twg, twu = T(x), T(wg), T(wu)
    assert fnmatch.fnmatch(gated_variant(tt, tx, twg, twu, True), tile) and ("_w" in tile) == ("_w" in gated_variant(tt, tx, twg, twu, True))
    dg, du = (dh * u * (g >= 0)).astype(np.float64), (dh * np.maximum(g, 0)).astype(np.float64)
    wide_x, wide_g, wide_u = (a.astype(np.float64) for a in (x, wg, wu))
    want = (dg @ wide_g.T + du @ wide_u.T, wide_x.T @ dg, wide_x.T @ du, dg.sum(0), du.sum(0))
    size = (np.abs(dg) @ np.abs(wide_g).T + np.abs(du) @ np.abs(wide_u).T, np.abs(wide_x).T @ np.abs(dg), np.abs(wide_x).T @ np.abs(du),
            np.abs(dg).sum(0), np.abs(du).sum(0))
    assert max(a.max() for a in size) < 1 / U[dtype]  # (exact in any order)
    frames = [framed(tt, a.shape, dtype) for a in want]
    got = tt.gated_linear_backward(T(dh), tx, twg, twu, T(g), T(u), activation="relu", out=tuple(f[0] for f in frames))
    for name, a, b, f in zip(("dx", "dwg", "dwu", "dbg", "dbu"), got, want, frames):
        assert np.array_equal(a.to_numpy().astype(np.float64), b), name
        assert f[1](), name
    none = tt.gated_linear_backward(T(dh), tx, twg, twu, T(g), T(u), activation="relu", bias_grad=False)
    assert all(np.array_equal(a.to_numpy(), b) for a, b in zip(none[:3], want))


def test_gated_linear_shapes(tt):
    r = rng_of(11)
    x, wg, wu, bg, bu, _ = gated_data(r, np.float32, 24, 40, 36)
    T = tt.Tensor.from_numpy
    flat = tt.gated_linear(T(x), T(wg), T(wu), T(bg), T(bu)).to_numpy()
    three = tt.gated_linear(T(x.reshape(2, 12, 40)), T(wg), T(wu), T(bg), T(bu))
    assert three.shape == (2, 12, 36) and np.array_equal(three.to_numpy().reshape(24, 36), flat)
    one = tt.gated_linear(T(x[0]), T(wg), T(wu), T(bg), T(bu))
    assert one.shape == (36,)
    g, u = gated_reference(x[:1], wg, wu, bg, bu, "silu")
    assert np.allclose(one.to_numpy(), (act_of(g, "silu")[0] * u)[0], rtol=1e-5, atol=1e-6)
    none = tt.gated_linear(T(x[:0]), T(wg), T(wu))
    assert none.shape == (0, 36)
    e = T(np.zeros((0, 36), np.float32))
    grads = tt.gated_linear_backward(e, T(x[:0]), T(wg), T(wu), e, e)
    assert grads[0].shape == (0, 40) and all(np.all(t.to_numpy() == 0) for t in grads[1:])


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_gated_linear_whole_numbers_and_infinities(tt, rows):
    """relu on whole numbers is exact (no term of the sums is lost or taken twice); an infinity reaches its row alone."""
    r = rng_of(rows, 5)
    x, wg, wu = (r.integers(-3, 4, s).astype(np.float32) for s in ((rows, 72), (72, 132), (72, 132)))
    dh = r.integers(-2, 3, (rows, 132)).astype(np.float32)
    T = tt.Tensor.from_numpy
    h, g, u = tt.gated_linear(T(x), T(wg), T(wu), activation="relu", save=True)
    wantg, wantu = x @ wg, x @ wu
    assert np.array_equal(g.to_numpy(), wantg) and np.array_equal(u.to_numpy(), wantu)
    assert np.array_equal(h.to_numpy(), np.maximum(wantg, 0) * wantu)
    got = tt.gated_linear_backward(T(dh), T(x), T(wg), T(wu), g, u, activation="relu")
    dg, du = (dh * wantu * (wantg >= 0)).astype(np.float64), (dh * np.maximum(wantg, 0)).astype(np.float64)
    want = (dg @ wg.T + du @ wu.T, x.T @ dg, x.T @ du, dg.sum(0), du.sum(0))
    assert max(np.abs(w).max() for w in want) < 2 ** 24
    for a, w in zip(got, want):
        assert np.array_equal(a.to_numpy().astype(np.float64), w)
    bad = x.copy()
    bad[rows // 2, 3] = np.inf
    h2 = tt.gated_linear(T(bad), T(wg), T(wu), activation="relu").to_numpy()
    keep = np.arange(rows) != rows // 2
    assert np.array_equal(h2[keep], h.to_numpy()[keep]) and not np.isfinite(h2[rows // 2]).all()


# ---- the distillation loss -----------------------------------------------------------------------------------------------


def distill_reference(z, ids, t_logit, temp, w):
    """loss, gradient, and what their tolerances need, in 64 bits."""
    z, t_logit = z.astype(np.float64), t_logit.astype(np.float64)
    rows, cols = z.shape
    loss, grad, rel = np.zeros(rows), np.zeros((rows, cols)), np.zeros((rows, cols))
    lt = np.zeros(rows)
    for r in range(rows):
        ok = (ids[r] >= 0) & (ids[r] < cols)
        t = np.where(ok, t_logit[r], -np.inf)
        if w[r] == 0 or not (np.any(t > -np.inf) or np.any(np.isnan(t))):
            continue
        with np.errstate(invalid="ignore", divide="ignore"):
            xt, xz = (t - t.max()) / temp, (z[r] - z[r].max()) / temp
            p, q = np.exp(xt), np.exp(xz)
            p, lq = p / p.sum(), xz - np.log(q.sum())
            q = q / q.sum()
            some = p != 0
            terms = p[some] * (np.log(p[some]) - lq[ids[r][some]])
            loss[r] = w[r] * temp ** 2 * terms.sum()
            share = np.zeros(cols)
            np.add.at(share, ids[r][ok], p[ok])
            grad[r] = w[r] * temp * (q - share)
            # relative errors, in u: of an exponential 4 |x| + 4 (the difference, the factor, the product; two of the
            # function), of a sum the mean of its terms' and a rounding a level
            eq, ep = np.where(q > 0, 4 * np.abs(xz) + 4, 0), np.where(p > 0, 4 * np.abs(np.where(np.isfinite(xt), xt, 0)) + 4, 0)
            sq, sp = (q * eq).sum() + cols / 64 + 24, (p * ep).sum() + 28
            share_err = np.zeros(cols)
            np.add.at(share_err, ids[r][ok], (p * (ep + sp + 4 + len(p)))[ok])
            rel[r] = w[r] * temp * (q * (eq + sq + 4) + share_err)
            fin = np.isfinite(terms)
            lt[r] = w[r] * temp ** 2 * ((np.abs(np.log(p[some]) - lq[ids[r][some]]) + 1) * p[some] * (ep[some] + sp + 4))[fin].sum() + w[r] * temp ** 2 * sq
    return loss.sum(), grad, rel, lt.sum() + np.abs(loss[np.isfinite(loss)]).sum() * 4


def check_distill(tt, z, ids, t_logit, temp, w, dtype, tz=None, index=np.int64):
    u = U[dtype]
    rows, cols = z.shape
    weight = np.full(rows, 1 / max(rows, 1)) if w is None else w.astype(np.float64)
    loss, grad, rel, lt = distill_reference(z, ids, t_logit, temp, weight)
    T = tt.Tensor.from_numpy
    out = framed(tt, (1,), dtype), framed(tt, (rows, cols), dtype)
    args = (tz if tz is not None else T(z), T(ids.astype(index)), T(t_logit))
    kw = dict(temperature=temp, row_weight=T(w) if w is not None else None)
    got = tt.distill_loss(*args, out=(out[0][0], out[1][0]), **kw)
    a, g = got[0].to_numpy()[0], got[1].to_numpy().astype(np.float64)
    assert out[0][1]() and out[1][1]()
    fin = np.isfinite(grad)
    assert np.array_equal(np.isnan(g), np.isnan(grad))
    assert np.all(np.abs(g[fin] - grad[fin]) <= u * rel[fin] + 4 * np.finfo(dtype).tiny), np.max(np.abs(g[fin] - grad[fin]) - u * rel[fin])
    if np.isfinite(loss):
        assert abs(a - loss) <= u * lt + u * abs(loss) + np.finfo(dtype).tiny, (a, loss, u * lt)
    else:
        assert (np.isnan(a) and np.isnan(loss)) or a == loss
    again = tt.distill_loss(*args, **kw)
    assert np.array_equal(again[0].to_numpy(), got[0].to_numpy(), equal_nan=True) and np.array_equal(again[1].to_numpy(), got[1].to_numpy(), equal_nan=True)
    return g


def distill_data(r, rows, cols, top, dtype):
    z = (r.normal(0, 2, (rows, cols))).astype(dtype)
    ids = np.stack([r.permutation(cols)[:top] if top <= cols else r.integers(0, cols, top) for _ in range(rows)]) if rows else np.zeros((0, top), np.int64)
    return z, ids, r.normal(2, 2, (rows, top)).astype(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols, top", [(1, 1, 1), (3, 2, 2), (5, 3, 1), (4, 10, 4), (130, 10, 10), (7, 17, 5), (3, 64, 8), (9, 65, 33), (2, 257, 64),
                                             (5, 1000, 100), (3, 1024, 7), (3, 1025, 64), (2, 2051, 300), (6, 4096, 64), (3, 8191, 1), (2, 8200, 1024),
                                             (2, 16390, 16), (1, 33001, 128), (3, 65537, 70), (2, 98305, 33), (2, 90000, 1024), (1, 150001, 300), (1, 131073, 64), (140, 5000, 12), (2, 200003, 9),
                                             (300, 2000, 3), (0, 8, 2), (2, 3, 300),
                                             (5, 1, 1024), (3, 70, 1000), (4, 2, 65), (3, 64, 64), (3, 63, 257), (2, 1024, 256), (2, 900, 257)])
def test_distill_loss(tt, dtype, rows, cols, top):
    r = rng_of(rows, cols, top)
    z, ids, t = distill_data(r, rows, cols, top, dtype)
    check_distill(tt, z, ids, t, 1.0 if cols % 2 else 2.5, None, dtype, index=np.int32 if top % 2 else np.int64)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows, cols, top", [(r, 40, 3) for r in (1, 3, 4, 5, 63, 64, 65)] + [(r, 700, 20) for r in (1, 2, 8, 9, 16, 17)] +
                         [(1, 700, 40), (2, 700, 40), (1, 50003, 70), (1, 90001, 70)])
def test_distill_loss_of_one_workgroup_or_more(tt, dtype, rows, cols, top):
    """Row counts on both sides of what one workgroup takes (it adds the loss up itself), with rows that do not count."""
    r = rng_of(rows, cols, top, "one")
    z, ids, t = distill_data(r, rows, cols, top, dtype)
    check_distill(tt, z, ids, t, 2.0, None, dtype)
    if rows > 1:
        ids[rows - 1] = -1                              # nothing in the last row, and no weight for the first
        w = r.random(rows).astype(dtype)
        w[0] = 0
        check_distill(tt, z, ids, t, 1.0, w, dtype)
    else:
        check_distill(tt, z, ids, t, 1.0, np.zeros(1, dtype), dtype)
        ids[0] = -1
        check_distill(tt, z, ids, t, 1.0, None, dtype)


@pytest.mark.parametrize("dtype, rows, cols", [(np.float32, 140, 60001), (np.float32, 130, 98309), (np.float32, 140, 131072), (np.float32, 129, 200003),
                                               (np.float64, 131, 65538), (np.float64, 129, 100001), (np.float32, 1600, 33000), (np.float32, 400, 131071),
                                               (np.float64, 700, 37001), (np.float32, 15000, 3501)])
def test_distill_loss_many_long_rows(tt, dtype, rows, cols):
    """Rows that fill a workgroup's registers and more, and matrices beyond the caches: three rows' data over and over."""
    r = rng_of(rows, cols)
    top = 20
    z, ids, t = distill_data(r, 3, cols, top, dtype)
    of = np.arange(rows) % 3
    w = (r.integers(0, 3, rows) / rows).astype(dtype)
    _, grad, rel, _ = distill_reference(z, ids, t, 2.0, np.ones(3))
    T = tt.Tensor.from_numpy
    loss, got = tt.distill_loss(T(z[of]), T(ids[of]), T(t[of]), temperature=2.0, row_weight=T(w))
    each = [distill_reference(z[k:k + 1], ids[k:k + 1], t[k:k + 1], 2.0, np.ones(1)) for k in range(3)]
    got = got.to_numpy()
    for k in range(3):
        at = np.flatnonzero(of == k)
        first = {}
        for i in at:     # equal rows and weights give equal bits
            assert np.array_equal(first.setdefault(w[i], got[i]), got[i])
        for weight, g in first.items():
            assert np.all(np.abs(g - weight * grad[k]) <= U[dtype] * (weight * rel[k] + 2 * np.abs(weight * grad[k])) + 1e-300)
    want = sum(each[of[i]][0] * float(w[i]) for i in range(rows))
    assert abs(loss.to_numpy()[0] - want) <= U[dtype] * (sum(each[of[i]][3] * float(w[i]) for i in range(rows)) + abs(want))


def test_distill_loss_from_two_threads(tt):
    """Calls that want different amounts of LDS of one kernel, from two threads with a stream each: the results of calls alone."""
    import ctypes
    import threading
    r = rng_of("threads")
    T, capi, lib = tt.Tensor.from_numpy, tt._capi, tt._capi.lib
    rows, calls, failed = 140, [], []
    for cols, top in ((66000, 5), (90000, 900)):     # 1024 lanes with 16 vectors each, and 1 or 6 vectors of LDS
        z, ids, t = distill_data(r, rows, cols, top, np.float32)
        ops = [T(z), T(ids.astype(np.int32)), T(t)]
        want = [x.to_numpy() for x in tt.distill_loss(*ops)]
        size = ctypes.c_size_t()
        assert lib.ttamd_distill_loss_workspace(capi.F32, rows, cols, top, ctypes.byref(size)) == capi.OK
        outs = [tt.Tensor.empty((1,), capi.F32), tt.Tensor.empty((rows, cols), capi.F32), tt.Tensor.empty((size.value // 4,), capi.F32)]
        stream = tt.graph.Stream(non_blocking=True)
        z, ids, t, loss, grad, ws = (x.storage.ptr for x in ops + outs)
        args = (0, capi.F32, capi.I32, rows, cols, top, z, cols, ids, t, None, 1.0, loss, grad, ws, size.value, stream.handle)
        calls.append((ops, outs, want, stream, args))

    def work(args):
        for _ in range(20):
            if lib.ttamd_distill_loss(*args) != capi.OK:
                failed.append(capi.last_error())

    threads = [threading.Thread(target=work, args=(c[-1],)) for c in calls]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
    for ops, (loss, grad, _), want, stream, _ in calls:
        stream.synchronize()
        assert np.array_equal(loss.to_numpy(), want[0]) and np.array_equal(grad.to_numpy(), want[1])
        stream.close()


def test_distill_loss_of_millions_of_rows(tt):
    """More rows than one launch takes."""
    rows, cols = (1 << 21) + 37, 3
    r = rng_of(rows)
    z, t = r.normal(0, 1, (rows, cols)).astype(np.float32), r.normal(0, 1, (rows, 2)).astype(np.float32)
    ids = np.stack([r.integers(0, cols, rows), r.integers(-1, cols, rows)], 1).astype(np.int32)
    T = tt.Tensor.from_numpy
    w = np.full(rows, 1.0, np.float32)
    _, got = tt.distill_loss(T(z), T(ids), T(t), row_weight=T(w))
    q = np.exp(z.astype(np.float64))
    q /= q.sum(1, keepdims=True)
    p = np.where(ids >= 0, np.exp(t.astype(np.float64)), 0)
    p /= p.sum(1, keepdims=True)
    for k in range(2):
        ok = ids[:, k] >= 0
        q[np.flatnonzero(ok), ids[ok, k]] -= p[ok, k]
    # (exponentials of arguments up to 12: 52 u, the sums and quotients of three and two terms some ten more, twice)
    assert np.max(np.abs(got.to_numpy() - q)) <= 150 * U[np.float32]
    # the loss of rows at the launches' ends, with all the others masked
    some = np.array([0, 5, (1 << 21) - 1, 1 << 21, (1 << 21) + 1, rows - 2, rows - 1])
    w[:] = 0
    w[some] = 1
    loss, _ = tt.distill_loss(T(z), T(ids), T(t), row_weight=T(w))
    want, _, _, rel = distill_reference(z[some], ids[some], t[some], 1.0, np.ones(len(some)))
    assert abs(loss.to_numpy()[0] - want) <= U[np.float32] * (rel + 2 * abs(want))
    w[:] = 0
    w[some] = 1 / 64
    half, _ = tt.distill_loss(T(z), T(ids), T(t), row_weight=T(w))
    assert half.to_numpy()[0] == loss.to_numpy()[0] / 64


# sizes of every way through the operator: tiny rows, a wave, workgroups of several sizes, rows cut into parts
MASK_SIZES = [(6, 12), (6, 300), (6, 3001), (6, 20000), (150, 9000), (6, 90001), (130, 70001)]


@pytest.mark.parametrize("rows, cols, large, low", [(130, (1 << 22) + 3, 1 << 16, 18.2), (1, (1 << 27) + 5, 1 << 12, 24.1)])
def test_distill_sums_over_millions_of_columns(tt, rows, cols, large, low):
    """`large` logits of 0 and millions of logits whose exponential 2^-low is too small to count beside what a lane has added up in
    32 bits, but which together are 2e-4 and 2e-3 of the sum.  Rows of weight 0 hold whatever the memory held."""
    T, u = tt.Tensor, U[np.float32]
    z = np.full(cols, -low * np.log(2), np.float32)
    z[:large] = 0
    ids, t_logit = np.array([5, 70000, cols - 1]), np.array([1.0, 0.5, -1.0], np.float32)
    where = sorted({0, rows // 2, rows - 1})
    weight = np.zeros(rows, np.float32)
    weight[where] = [0.25, 0.5, 1.0][:len(where)]
    whole, one = T.empty((rows, cols), tt._capi.F32), T.from_numpy(z)
    for r in where:
        T(whole.storage, whole.dtype, (cols,), (1,), r * cols).assign(one)
    loss, grad = tt.distill_loss(whole, T.from_numpy(np.tile(ids, (rows, 1))), T.from_numpy(np.tile(t_logit, (rows, 1))), row_weight=T.from_numpy(weight))
    small = float(z[-1])
    log_total = np.log(large + (cols - large) * np.exp(small))
    p = np.exp(t_logit.astype(np.float64))
    p /= p.sum()
    lq = z[ids].astype(np.float64) - log_total
    # Relative roundings: an exponential 4 |x| + 4; the sum 3 a vector, 8 vectors kept in LDS (the ones before them add up exactly),
    # 10 of the tree, a conversion, or 16 and 10 of a part, a product: below 32;
    # the quotient, the factor and the product 4 more; p of 3 slots 4 |t| + 4 each, 3 for their sum, the quotient, the weight: below 40.
    q_tol = lambda x: (4 * np.abs(x) + 4 + 32 + 4) * u  # noqa: E731
    for r in where:
        w = float(weight[r])
        got = T(grad.storage, grad.dtype, (cols,), (1,), r * cols).contiguous().to_numpy().astype(np.float64)
        for j, i in enumerate(ids):
            q = np.exp(lq[j])
            assert abs(got[i] - w * (q - p[j])) <= w * (q * q_tol(z[i]) + 40 * u * p[j])
        got = np.delete(got, ids)
        for part, x in ((got[:large - 1], 0.0), (got[large - 1:], small)):
            assert np.all(np.abs(part - w * np.exp(x - log_total)) <= w * np.exp(x - log_total) * q_tol(x))
    terms = p * (np.log(p) - lq)
    want = weight.sum(dtype=np.float64) * terms.sum()
    tol = weight.sum(dtype=np.float64) * u * ((p * (np.abs(np.log(p) - lq) + 1)).sum() * 40 + 32) + 4 * u * abs(want)
    assert abs(loss.to_numpy()[0] - want) <= tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", MASK_SIZES)
def test_distill_masks(tt, dtype, rows, cols):
    r = rng_of(rows, cols, 2)
    top = 7
    z, ids, t = distill_data(r, rows, cols, top, dtype)
    w = r.random(rows).astype(dtype)
    w[1] = 0
    z[1] = np.nan                                       # weighs nothing: never looked at
    ids[2] = [-1, cols, -5, cols + 7, 1 << 30, -(1 << 31), cols]  # no slot counts
    t[3] = -np.inf                                      # nothing left of the teacher
    ids[4, :3] = ids[4, 3]                              # one column several times
    ids[0, 2], t[0, 3] = -1, -np.inf                    # padding and an impossible column among others
    z[5] = np.finfo(dtype).min                          # the lowest value everywhere but at a few columns
    z[5, ids[5]] = r.normal(0, 1, top)
    z[0, 5:9] = -np.inf                                 # words the student may not say
    ids[0, :] = np.where((ids[0] >= 5) & (ids[0] < 9), 0, ids[0])
    g = check_distill(tt, z, ids, t, 2.0, w, dtype, index=np.int32)
    assert np.all(g[1] == 0) and np.all(g[2] == 0) and np.all(g[3] == 0) and np.all(g[0, 5:9] == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", MASK_SIZES)
def test_distill_infinities(tt, dtype, rows, cols):
    r = rng_of(rows, cols, 3)
    z, ids, t = distill_data(r, rows, cols, 4, dtype)
    z[0] = -np.inf                                      # no column is possible: not a number, in this row alone
    z[1, cols // 2] = np.inf
    z[2, cols - 1] = np.nan
    z[3, : cols - 2] = -np.inf                          # all but the last two columns impossible
    ids[3] = cols - 1
    g = check_distill(tt, z, ids, t, 1.0, None, dtype)
    assert np.isnan(g[:3]).all() and np.isfinite(g[3:]).all()
    # the teacher wants a word that the student may not say: an infinite loss, a finite gradient
    z, ids, t = distill_data(r, rows, cols, 4, dtype)
    z[1, ids[1, 0]] = -np.inf
    check_distill(tt, z, ids, t, 1.0, None, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(5, 10), (5, 1003), (4, 6001), (3, 40002)])
def test_distill_rows_apart(tt, dtype, rows, cols):
    """Logits that are part of a wider matrix, beginning off every boundary."""
    r = rng_of(rows, cols, 4)
    z, ids, t = distill_data(r, rows, cols, 5, dtype)
    wide = np.full((rows, cols + 5), np.nan, dtype)
    wide[:, 3:3 + cols] = z
    whole = tt.Tensor.from_numpy(wide)
    check_distill(tt, z, ids, t, 1.5, None, dtype, tz=tt.Tensor(whole.storage, whole.dtype, z.shape, (cols + 5, 1), 3))
    turned = tt.Tensor.from_numpy(np.ascontiguousarray(z.T)).permute(1, 0)  # copied
    check_distill(tt, z, ids, t, 1.5, None, dtype, tz=turned)


# ---- gradients against differences, a whole step, graphs --------------------------------------------------------------------


def slope_of(f, args, k, r, eps=1e-6):
    d = r.normal(0, 1, args[k].shape)
    up, down = list(args), list(args)
    up[k], down[k] = args[k] + eps * d, args[k] - eps * d
    return (f(*up) - f(*down)) / (2 * eps), d


def student_step(tt, table, wg, wu, wo, ids, t_ids, t_logit, scale):
    """Loss and gradients of tokens -> embedding -> gated pair -> output layer -> distillation loss; the table's gradient is
    added onto its use as an output layer (logits over the vocabulary through a projection wo and the table)."""
    x = tt.embedding(ids, table, scale=scale)
    h, g, u = tt.gated_linear(x, wg, wu, activation="silu", save=True)
    y = tt.linear(h, wo)
    logits = tt.linear(y, table.permute(1, 0))
    loss, dlogits = tt.distill_loss(logits, t_ids, t_logit, temperature=2.0)
    dtable = tt.matmul(dlogits.permute(1, 0), y)                  # of the output layer, [vocab, dim]
    dy = tt.matmul(dlogits, table)
    dh, dwo, _ = tt.linear_backward(dy, h, wo, bias_grad=False)
    dx, dwg, dwu, _, _ = tt.gated_linear_backward(dh, x, wg, wu, g, u, activation="silu", bias_grad=False)
    tt.embedding_backward(dx, ids, table.size(0), scale=scale, out=dtable, accumulate=True)
    return loss, dtable, dwg, dwu, dwo


def student_data(r, dtype, count=60, vocab=50, dim=24, hidden=40, top=5):
    n = lambda *s: r.normal(0, 1, s).astype(dtype)  # noqa: E731
    return dict(table=n(vocab, dim) * dtype(0.5), wg=n(dim, hidden) * dtype(0.2), wu=n(dim, hidden) * dtype(0.2), wo=n(hidden, dim) * dtype(0.2)), \
        dict(ids=r.integers(0, vocab, count).astype(np.int64), t_ids=np.stack([r.permutation(vocab)[:top] for _ in range(count)]).astype(np.int32), t_logit=n(count, top))


def student_loss(table, wg, wu, wo, ids, t_ids, t_logit, scale):
    x = table[ids] * scale
    g, u = x @ wg, x @ wu
    logits = (act_of(g, "silu")[0] * u) @ wo @ table.T
    return distill_reference(logits, t_ids, t_logit, 2.0, np.full(len(ids), 1 / len(ids)))[0]


def test_student_step_gradients(tt):
    """The operators together, as a training step uses them: loss and all gradients against differences of the formula."""
    r = rng_of(21)
    weights, data = student_data(r, np.float64)
    T = tt.Tensor.from_numpy
    got = student_step(tt, **{k: T(v) for k, v in {**weights, **data}.items()}, scale=1.5)
    f = lambda table, wg, wu, wo: student_loss(table, wg, wu, wo, **data, scale=1.5)  # noqa: E731
    args = [weights[k] for k in ("table", "wg", "wu", "wo")]
    assert abs(got[0].to_numpy()[0] - f(*args)) <= 1e-12 * abs(f(*args))
    for k, grad in enumerate(got[1:]):
        want, d = slope_of(f, args, k, r)
        # central differences: eps^2 of the third derivative and 1e-16 / eps of the value
        assert abs((grad.to_numpy() * d).sum() - want) <= 1e-7 * max(1, abs(want)), k


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_gated_gradients_against_differences(tt, act):
    r = rng_of(22)
    x, wg, wu, bg, bu, dh = gated_data(r, np.float64, 6, 10, 14)

    def f(x, wg, wu, bg, bu):
        g, u = gated_reference(x, wg, wu, bg, bu, act)
        return (act_of(g, act)[0] * u * dh).sum()

    T = tt.Tensor.from_numpy
    _, g, u = tt.gated_linear(T(x), T(wg), T(wu), T(bg), T(bu), activation=act, save=True)
    got = tt.gated_linear_backward(T(dh), T(x), T(wg), T(wu), g, u, activation=act)
    for k, grad in enumerate(got):
        want, d = slope_of(f, [x, wg, wu, bg, bu], k, r)
        assert abs((grad.to_numpy() * d).sum() - want) <= 1e-7 * max(1, abs(want)), k


def test_student_step_as_a_graph(tt):
    """The whole step captured once and replayed on fresh inputs, with eager work in between: the same bits as eager runs.
    A second graph of the same step, replayed in turn, has workspaces of its own."""
    r = rng_of(23)
    weights, data = student_data(r, np.float32, count=300, vocab=700, dim=64, hidden=96, top=9)
    T = tt.Tensor.from_numpy
    be = tt.get_backend(tt.kAMD)
    fixed = {k: T(v) for k, v in weights.items()}
    streams = [tt.graph.Stream(), tt.graph.Stream(non_blocking=True)]
    graphs, inputs = [], []
    try:
        for s in streams:
            inp = {k: T(v) for k, v in data.items()}
            be.synchronize(0)
            inputs.append(inp)
            graphs.append(tt.graph.Graph(s, lambda inp=inp: student_step(tt, **fixed, **inp, scale=1.25)))
        for replay in range(3):
            fresh = [student_data(rng_of(40 + replay, j), np.float32, count=300, vocab=700, dim=64, hidden=96, top=9)[1] for j in range(2)]
            for inp, new, g in zip(inputs, fresh, graphs):
                for k, v in new.items():
                    g.copy_in(inp[k], v)
            be.synchronize(0)
            for g in graphs:
                g.launch()      # both in flight together
            for s in streams:
                s.synchronize()
            for new, g in zip(fresh, graphs):
                got = [t.to_numpy() for t in g.outputs]
                eager = [t.to_numpy() for t in student_step(tt, **fixed, **{k: T(v) for k, v in new.items()}, scale=1.25)]
                for a, b in zip(got, eager):
                    assert np.array_equal(a, b)
            be.synchronize(0)
    finally:
        for g in graphs:
            g.close()
        for s in streams:
            s.close()


def test_on_another_stream(tt):
    """The operators follow on_stream(): enqueued there, in order with what the stream did before."""
    r = rng_of(24)
    weights, data = student_data(r, np.float32)
    T = tt.Tensor.from_numpy
    dev = {k: T(v) for k, v in {**weights, **data}.items()}
    want = [t.to_numpy() for t in student_step(tt, **dev, scale=1.0)]
    stream = tt.graph.Stream(non_blocking=True)
    try:
        tt.get_backend(tt.kAMD).synchronize(0)
        got = stream.run(lambda: student_step(tt, **dev, scale=1.0))
        stream.synchronize()
        for a, b in zip(want, got):
            assert np.array_equal(a, b.to_numpy())
        del got
    finally:
        stream.close()
