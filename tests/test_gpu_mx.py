"""The MX entry points against the 64-bit statement of mx_ref.

Bars. Quantised codes, scales, dequantised values, sums and sorted rows are
exact. A norm is the exact value rounded once: half a step, 2^-24 relative.
Products are tested for equality on operands whose sums are exact in fp32 in
any order (few-bit elements and scales close together, so that every partial
sum is a whole number of quanta below 2^24), which leaves no tolerance for a
misplaced row, column, block or scale; on ordinary values each product carries
at most one rounding per term, K 2^-23 sum|x w|. SwiGLU's 8-bit result is off
the exact value by half an element step, plus the fp32 chain before it: expf
and the quotient 2 ulp each, four more roundings, under 8 * 2^-24 * 2 in all.
"""

from __future__ import annotations

import numpy as np
import pytest

import mx_ref as R
from conftest import assert_bitexact
from qw3_b200 import inputs as I

pytestmark = pytest.mark.gpu

FP8, FP4 = R.FP8, R.FP4
F32, F16 = 0, 1


class Bufs:
    def __init__(self, ds3):
        self.d, self.all = ds3, []

    def up(self, a):
        if a is None:
            return None
        self.all.append(self.d.upload(np.ascontiguousarray(a)))
        return self.all[-1]

    def shifted(self, a, by):
        """The array at `by` bytes into a fresh allocation."""
        a = np.ascontiguousarray(a)
        base = self.up(np.zeros(a.nbytes + by, np.uint8))
        v = self.d.buffer_view(base, by, a.nbytes)
        self.all.append(v)
        assert self.d.buffer_write(v, 0, a) == 0
        return v

    def down(self, b, dtype, shape):
        return self.d.download(b, dtype, shape)


@pytest.fixture
def B(ds3):
    b = Bufs(ds3)
    yield b
    for x in b.all:
        x.free()
    assert ds3.device_errors() == 0


# ------------------------------------------------------ quantise, dequantise
def same_values(got, want):
    """Bit-exact fp32 values, NaN in the same places."""
    want = want.astype(np.float32)
    assert (np.isnan(got) == np.isnan(want)).all()
    assert_bitexact(np.where(np.isnan(got), 0, got), np.where(np.isnan(want), 0, want), "values")


def awkward(rows, cols, dtype, seed):
    """Rows with ordinary values, exact ties, zeros, tiny and huge blocks (the
    huge fp16 ones hold infinities)."""
    x = I.normal(seed, (rows, cols), 0.0, 3.0)
    b = x.reshape(-1, 32)
    kinds = np.arange(b.shape[0]) % 8
    b[kinds == 1] = 0.0
    b[kinds == 2] = -0.0
    ties = np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 17.0, 19.0, 25.0, 27.0, -0.25, -2.5, -5.0, 7.9],
                            np.float32), 2)
    b[kinds == 3] = ties
    b[kinds == 4] *= np.float32(1e-41 if dtype == np.float32 else 1e-7)
    b[kinds == 5] *= np.float32(1e37 if dtype == np.float32 else 1e4)
    b[kinds == 6] = np.where(np.arange(32) == 7, np.float32(463.9), b[kinds == 6])  # past 448: saturates
    with np.errstate(over="ignore"):
        return x.astype(dtype)


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (7, 1024), (129, 2048), (1000, 160)])
def test_quantize_and_back(ds3, B, fmt, dtype, rows, cols):
    x = awkward(rows, cols, dtype, rows + cols)
    q = B.up(np.full(rows * cols // (2 if fmt == FP4 else 1) + 16, 0xA5, np.uint8))
    s = B.up(np.full(rows * cols // 32 + 16, 0xA5, np.uint8))
    assert ds3.mx_quantize(B.up(x), F32 if dtype == np.float32 else F16, q, s, fmt, rows, cols) == 0, ds3.last_error()
    wq, ws = R.encode(x, fmt)
    got_q, got_s = B.down(q, np.uint8, (wq.size + 16,)), B.down(s, np.uint8, (ws.size + 16,))
    assert_bitexact(got_s[:-16].reshape(ws.shape), ws, "scales")
    assert_bitexact(got_q[:-16].reshape(wq.shape), wq, "elements")
    assert (got_q[-16:] == 0xA5).all() and (got_s[-16:] == 0xA5).all()
    out = B.up(np.full((rows, cols), np.nan, np.float32))
    assert ds3.mx_dequantize(q, s, fmt, out, rows, cols) == 0
    want = R.decode(wq, ws, fmt)
    got = B.down(out, np.float32, (rows, cols))
    assert np.array_equal(want.astype(np.float32), want, equal_nan=True)  # every value is an fp32 value
    same_values(got, want)


@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_dequantize_every_code_and_scale(ds3, B, fmt):
    """All element codes at all scales, NaN ones included."""
    codes = np.tile(np.arange(256, dtype=np.uint8), 256).reshape(256, 256)
    q = codes if fmt == FP8 else R.pack4(codes & 15)
    s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 8, 1)
    out = B.up(np.zeros((256, 256), np.float32))
    assert ds3.mx_dequantize(B.up(q), B.up(s), fmt, out, 256, 256) == 0
    got = B.down(out, np.float32, (256, 256))
    with np.errstate(over="ignore"):
        want = R.decode(q, s, fmt).astype(np.float32)
    same_values(got, want)


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_quantize_nonfinite_block_is_nan(ds3, B, fmt, bad):
    x = I.normal(5, (4, 64))
    x[1, 40] = bad
    q, s, out = B.up(np.zeros(256, np.uint8)), B.up(np.zeros(8, np.uint8)), B.up(np.zeros((4, 64), np.float32))
    assert ds3.mx_quantize(B.up(x), F32, q, s, fmt, 4, 64) == 0
    wq, ws = R.encode(x, fmt)
    assert ws[1, 1] == 255
    assert_bitexact(B.down(s, np.uint8, (4, 2)), ws, "scales")
    assert_bitexact(B.down(q, np.uint8, wq.shape), wq, "elements")
    assert ds3.mx_dequantize(q, s, fmt, out, 4, 64) == 0
    got = B.down(out, np.float32, (4, 64))
    assert np.isnan(got[1, 32:]).all() and np.isfinite(np.delete(got.reshape(8, 32), 3, 0)).all()


def test_quantize_no_rows(ds3, B):
    b = B.up(np.zeros(64, np.uint8))
    c = B.up(np.zeros(64, np.uint8))
    d = B.up(np.zeros(64, np.uint8))
    assert ds3.mx_quantize(b, F32, c, d, FP8, 0, 32) == 0
    assert ds3.mx_dequantize(b, c, FP8, d, 0, 32) == 0


# ---------------------------------------------------------------------- norm
def run_norm(ds3, B, x, r, w, eps=1e-6, alias=None, norm_out=True, sum_out=True):
    rows, n = x.shape
    xb, rb, wb = B.up(x), B.up(r), B.up(w)
    sb = {"x": xb, "r": rb}.get(alias) if alias in ("x", "r") else B.up(np.zeros_like(x)) if sum_out else None
    nb = xb if alias == "norm" else B.up(np.zeros_like(x)) if norm_out else None
    q, sc = B.up(np.zeros((rows, n), np.uint8)), B.up(np.zeros((rows, n // 32), np.uint8))
    assert ds3.add_rms_norm_mx(xb, rb, wb, sb, nb, q, sc, n, rows, eps) == 0, ds3.last_error()
    get = lambda b: None if b is None else B.down(b, np.float32, x.shape)  # noqa: E731
    return get(sb), get(nb), B.down(q, np.uint8, (rows, n)), B.down(sc, np.uint8, (rows, n // 32))


def check_norm(x, r, w, eps, got):
    s, norm, q, sc = got
    ws, wn = R.add_norm(x, r, w, eps)
    if s is not None:
        assert_bitexact(s, ws, "sum")
    if norm is not None:
        # rounded once: half a step of 2^-23, and the carried products' own 2^-45;
        # below the normal range a step is 2^-149 whatever the value
        assert (np.abs(norm - wn) <= np.abs(wn) * 2.0**-24 * (1 + 2.0**-18) + 2.0**-150).all()
    wq, wsc = R.encode(wn.astype(np.float32), FP8)
    assert_bitexact(sc, wsc, "scales")
    assert_bitexact(q, wq, "elements")


@pytest.mark.parametrize("rows,n", [(1, 32), (3, 96), (17, 768), (1, 2048), (64, 2048), (149, 2048), (1500, 2048),
                                    (33, 4096), (200, 992), (5, 8224), (3, 16384), (4000, 256)])
def test_norm(ds3, B, rows, n):
    x, r, w = I.normal(rows, (rows, n)), I.normal(rows + 1, (rows, n), 0.0, 2.0), I.gamma(n, 3)
    check_norm(x, r, w, 1e-6, run_norm(ds3, B, x, r, w))


@pytest.mark.parametrize("alias", ["x", "r", "norm"])
def test_norm_in_place(ds3, B, alias):
    x, r, w = I.normal(1, (700, 512)), I.normal(2, (700, 512)), I.gamma(512, 3)
    check_norm(x, r, w, 1e-6, run_norm(ds3, B, x, r, w, alias=alias))


def test_norm_optional_outputs(ds3, B):
    x, w = I.normal(1, (300, 640)), I.gamma(640, 3)
    check_norm(x, None, w, 1e-5, run_norm(ds3, B, x, None, w, eps=1e-5))
    check_norm(x, x, w, 1e-5, run_norm(ds3, B, x, x, w, eps=1e-5, norm_out=False, sum_out=False))


@pytest.mark.parametrize("rows,n", [(1000, 5120), (700, 8192), (1500, 8224), (470, 16384)])
@pytest.mark.parametrize("form", ["plain", "no residual", "x", "r", "norm"])
def test_norm_long_rows_many_per_warp(ds3, B, rows, n, form):
    """Rows staged in shared memory, two and more to each warp, so that every
    slot is used again: two slots up to 8192 elements, one past that. (Rows
    without a residual take half the space, and twice the warps fit.)"""
    rows *= 2 if form == "no residual" else 1
    x, r, w = I.normal(rows, (rows, n)), I.normal(rows + 1, (rows, n), 0.0, 2.0), I.gamma(n, 3)
    r = None if form == "no residual" else r
    alias = form if form in ("x", "r", "norm") else None
    check_norm(x, r, w, 1e-6, run_norm(ds3, B, x, r, w, alias=alias))


def test_norm_extreme_rows(ds3, B):
    """Zero rows, rows whose squares pass fp32's range either way."""
    x, w = I.normal(1, (6, 128)), I.gamma(128, 3)
    x[1] = 0.0
    x[2] *= np.float32(1e25)
    x[3] *= np.float32(1e-25)
    x[4, 5] = 3e38
    check_norm(x, None, w, 1e-6, run_norm(ds3, B, x, None, w))


@pytest.mark.parametrize("n", [128, 8224])
def test_norm_factors_out_of_range(ds3, B, n):
    """An inverse root past fp32's range (subnormal rows, eps 0) and weights
    that carry normed values past it: the exact value rounded once, infinite
    where that is."""
    x, w = I.normal(1, (3, n)), I.gamma(n, 3)
    x[1] *= np.float32(1e-40)
    w[64] = 3e38
    got = run_norm(ds3, B, x, None, w, eps=0.0)
    _, wn = R.add_norm(x, None, w, 0.0)
    with np.errstate(over="ignore"):
        want = wn.astype(np.float32)
    assert np.isinf(want[:, 64]).any() and np.isfinite(np.delete(want, 64, 1)).all()
    fin = np.isfinite(want)
    assert (got[1][~fin] == want[~fin]).all(), "infinities"
    assert (np.abs(got[1] - wn)[fin] <= np.abs(wn[fin]) * 2.0**-24 * (1 + 2.0**-18) + 2.0**-150).all()
    wq, ws = R.encode(want, FP8)
    assert_bitexact(got[3], ws, "scales")
    assert_bitexact(got[2], wq, "elements")


@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_norm_nonfinite_row(ds3, B, bad):
    """As the plain formula: an infinity makes its own place NaN and the rest
    of the row 0, a NaN the whole row; other rows are untouched."""
    x, w = I.normal(1, (3, 128)), I.gamma(128, 3)
    x[1, 70] = bad
    _, norm, q, sc = run_norm(ds3, B, x, None, w)
    _, wn = R.add_norm(x, None, w, 1e-6)
    assert (np.isnan(norm) == np.isnan(wn)).all()
    wq, ws = R.encode(wn.astype(np.float32), FP8)
    assert_bitexact(sc, ws, "scales")
    assert_bitexact(np.where(ws.repeat(32, 1) == 255, 0, q), np.where(ws.repeat(32, 1) == 255, 0, wq), "elements")
    assert (q.reshape(3, 4, 32)[ws == 255] == 0).all()


def test_norm_matches_add_rms_norm(ds3, B):
    """The fp32 norm agrees with add_rms_norm's within the two roundings more that one makes."""
    x, r, w = I.normal(1, (64, 2048)), I.normal(2, (64, 2048)), I.gamma(2048, 3)
    _, norm, _, _ = run_norm(ds3, B, x, r, w)
    s, o = B.up(np.zeros_like(x)), B.up(np.zeros_like(x))
    assert ds3.add_rms_norm(B.up(x), B.up(r), B.up(w), s, o, 2048, 64, 1e-6) == 0
    other = B.down(o, np.float32, x.shape)
    assert (np.abs(norm - other) <= 1e-5 * np.abs(other) + 1e-6).all()


# --------------------------------------------------------------- sorted rows
def run_rows(ds3, B, idx, E, shift=0):
    n = idx.size
    ib = B.shifted(idx, shift) if shift else B.up(idx)
    off, ent, row = B.up(np.full(E + 1, -7, np.int32)), B.up(np.full(n, -7, np.int32)), B.up(np.full(n, -7, np.int32))
    rc = ds3.moe_expert_rows(ib, off, ent, row, idx.shape[0], E, idx.shape[1])
    return rc, [B.down(b, np.int32, (k,)) for b, k in ((off, E + 1), (ent, n), (row, n))]


@pytest.mark.parametrize("T,E,K", [(1, 128, 8), (1, 1, 1), (3, 256, 8), (37, 64, 4), (512, 128, 8), (700, 256, 3),
                                   (5000, 60, 1), (8191, 128, 8), (8192, 40, 8), (8193, 40, 8),
                                   (30000, 250, 5)])
def test_expert_rows(ds3, B, T, E, K):
    idx = np.argsort(I.rng(T + E).random((T, E)), 1)[:, :K].astype(np.int32)
    rc, got = run_rows(ds3, B, idx, E)
    assert rc == 0, ds3.last_error()
    for g, w, name in zip(got, R.expert_rows(idx, E), ("offsets", "entries", "row_of")):
        assert_bitexact(g, w, name)


def test_expert_rows_unaligned_ids_one_expert_and_no_map(ds3, B):
    idx = np.full((333, 3), 5, np.int32)  # every entry to one expert
    rc, got = run_rows(ds3, B, idx, 9, shift=4)
    assert rc == 0
    for g, w in zip(got, R.expert_rows(idx, 9)):
        assert_bitexact(g, w)
    off, ent = B.up(np.zeros(10, np.int32)), B.up(np.zeros(999, np.int32))
    assert ds3.moe_expert_rows(B.up(idx), off, ent, None, 333, 9, 3) == 0
    assert_bitexact(B.down(ent, np.int32, (999,)), np.arange(999, dtype=np.int32))


def test_expert_rows_bad_ids(ds3, B):
    idx = I.rng(3).integers(0, 16, (50, 4)).astype(np.int32)
    idx[7, 2], idx[20, 0], idx[49, 3] = -1, 16, 1 << 30
    rc, (off, ent, row) = run_rows(ds3, B, idx, 16)
    assert rc == -1
    w_off, w_ent, w_row = R.expert_rows(idx, 16)
    assert_bitexact(off, w_off)
    assert_bitexact(ent[:197], w_ent)
    assert (ent[197:] == -7).all()
    assert_bitexact(row, w_row)


@pytest.mark.parametrize("n", [28 * 1024, 28 * 1024 + 1, 65536, 65537, 200003])
def test_expert_rows_many_entries_bad_ids_unaligned(ds3, B, n):
    """Sizes on both sides of the switch to clusters and of their chunks, ids
    out of range either way, and expert counts that leave a cluster part-filled."""
    idx = I.rng(n).integers(0, 19, (n, 1)).astype(np.int32)
    idx[[0, n // 2, n - 1]] = np.array([[19], [-1], [-(1 << 31)]], np.int32)
    idx[5::7] = 18  # a popular last expert
    rc, (off, ent, row) = run_rows(ds3, B, idx, 19, shift=4)
    assert rc == -1
    w_off, w_ent, w_row = R.expert_rows(idx, 19)
    assert_bitexact(off, w_off)
    assert_bitexact(ent[: len(w_ent)], w_ent)
    assert (ent[len(w_ent):] == -7).all()
    assert_bitexact(row, w_row)
    ib = B.up(np.full((n, 1), 3, np.int32))  # all to one, no map
    off, ent = B.up(np.zeros(10, np.int32)), B.up(np.zeros(n, np.int32))
    assert ds3.moe_expert_rows(ib, off, ent, None, n, 9, 1) == 0, ds3.last_error()
    assert_bitexact(B.down(off, np.int32, (10,)), np.array([0] * 4 + [n] * 6, np.int32))
    assert_bitexact(B.down(ent, np.int32, (n,)), np.arange(n, dtype=np.int32))


def test_expert_rows_no_tokens(ds3, B):
    off = B.up(np.full(5, 9, np.int32))
    e = B.up(np.zeros(4, np.int32))
    assert ds3.moe_expert_rows(B.up(np.zeros(4, np.int32)), off, e, None, 0, 4, 8) == 0
    assert_bitexact(B.down(off, np.int32, (5,)), np.zeros(5, np.int32))


# ---------------------------------------------------------- grouped products
def exact_rows(seed, rows, cols, fmt, spread=3):
    """MX rows whose products' sums are exact in fp32: elements 0, 1/2, 1, 2, 3
    and 4 of either sign, scales 2^-1 .. 2^1 (quantum 2^-4, so 2^-4 .. 64 per
    term and 4096 terms stay below 2^24 quanta)."""
    g = I.rng(seed)
    pool = np.array([0.0, 0.5, 1.0, 2.0, 3.0, 4.0, -0.5, -1.0, -2.0, -3.0, -4.0])
    t = R.table(fmt)
    code = np.array([int(np.flatnonzero((t == p) & (np.signbit(t) == np.signbit(p)))[0]) for p in pool], np.uint8)
    c = code[g.integers(0, len(pool), (rows, cols))]
    s = g.integers(126, 126 + spread, (rows, cols // 32)).astype(np.uint8)
    return (R.pack4(c) if fmt == FP4 else c), s


def ragged(seed, rows, E, empty=0.3):
    """offsets of E groups over `rows` rows, some empty."""
    g = I.rng(seed)
    p = g.random(E) * (g.random(E) > empty) + 1e-9
    return np.concatenate([[0], np.cumsum(g.multinomial(rows, p / p.sum()))]).astype(np.int32)


def run_matmul(ds3, B, x, xs, w, ws, fmt, off, n_rows, out, x_rows=None, x_div=1, out_rows=None):
    E, N, K = ws.shape[0], ws.shape[1], ws.shape[2] * 32
    ob = B.up(out)
    rc = ds3.moe_mx_matmul(B.up(x), B.up(xs), B.up(x_rows), x_div, B.up(off), B.up(w), B.up(ws), fmt, ob,
                           F16 if out.dtype == np.float16 else F32, B.up(out_rows), xs.shape[0], n_rows, E, K, N)
    return rc, B.down(ob, out.dtype, out.shape)


SHAPES = [
    # rows, experts, K, N
    (1, 1, 32, 1), (1, 4, 128, 32), (5, 3, 160, 100), (16, 2, 256, 128), (17, 1, 128, 129), (63, 1, 512, 64),
    (64, 1, 768, 256), (65, 1, 1024, 130), (130, 2, 2048, 64), (200, 60, 384, 200), (300, 256, 128, 36),
    (257, 2, 640, 96), (500, 3, 256, 257), (900, 3, 512, 128), (1300, 4, 4096, 48), (224, 1, 128, 128),
    (225, 1, 96, 31), (2000, 7, 224, 33),
]


@pytest.mark.parametrize("rows,E,K,N", SHAPES)
@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("mapped", [False, True])
def test_matmul_exact(ds3, B, rows, E, K, N, fmt, mapped):
    if fmt == FP4:
        K = -(-K // 128) * 128
    used = 3
    n_x = rows + 5 if not mapped else rows // 2 + 1
    x, xs = exact_rows(1, n_x, K, FP8)
    w, ws = exact_rows(2, E * N, K, fmt)
    w, ws = w.reshape(E, N, -1), ws.reshape(E, N, -1)
    off = ragged(3, rows, E)
    g = I.rng(4)
    x_rows = g.integers(0, n_x * used, rows).astype(np.int32) if mapped else None
    out_rows = g.permutation(rows + 7)[:rows].astype(np.int32) if mapped else None
    dtype = np.float16 if mapped and rows % 2 else np.float32
    out = np.full((rows + 7, N), -77.0, dtype)
    rc, got = run_matmul(ds3, B, x, xs, w, ws, fmt, off, rows, out, x_rows, used, out_rows)
    assert rc == 0, ds3.last_error()
    src = x_rows // used if mapped else np.arange(rows)
    y = R.grouped(R.decode(x, xs, FP8), R.decode(w, ws, fmt), off, src)
    want = out.copy()
    want[out_rows if mapped else np.arange(rows)] = y.astype(np.float32).astype(dtype)
    assert_bitexact(got, want, "out")


@pytest.mark.parametrize("rows,E,K,N", [(3000, 60, 640, 1700), (3000, 14, 768, 2000), (6000, 12, 1024, 1500),
                                        (9000, 40, 256, 1000)])
@pytest.mark.parametrize("mapped", [False, True])
def test_matmul_many_tiles_per_cta(ds3, B, rows, E, K, N, mapped):
    """Several tiles for every CTA, at each token width the launcher picks, so
    that the rings of stages wrap many times and across tiles."""
    x, xs = exact_rows(1, rows, K, FP8)
    w, ws = exact_rows(2, E * N, K, FP8)
    w, ws = w.reshape(E, N, -1), ws.reshape(E, N, -1)
    off = ragged(3, rows, E, 0.1)
    src = I.rng(4).permutation(rows).astype(np.int32) if mapped else None
    rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, off, rows, np.zeros((rows, N), np.float32), src)
    assert rc == 0, ds3.last_error()
    want = R.grouped(R.decode(x, xs, FP8), R.decode(w, ws, FP8), off, src if mapped else np.arange(rows))
    assert_bitexact(got, want.astype(np.float32), "out")


@pytest.mark.parametrize("rows,E", [(900, 20), (1500, 16), (3000, 12)])
@pytest.mark.parametrize("N", [1000, 1004, 1001])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shift", [0, 8])
def test_matmul_output_units(ds3, B, rows, E, N, dtype, shift):
    """Every way of storing output rows: whole 16-byte units of either type, and
    rows whose length or address is not a whole number of them; rows in any
    order, an x row out of range (zeros) and an output row out of range."""
    K = 256
    x, xs = exact_rows(1, rows, K, FP8)
    w, ws = exact_rows(2, E * N, K, FP4)
    off = ragged(3, rows, E, 0.1)
    g = I.rng(4)
    x_rows, out_rows = g.permutation(rows).astype(np.int32), g.permutation(rows).astype(np.int32)
    bad_x, bad_o = off[-1] // 2, off[-1] // 3
    x_rows[bad_x], out_rows[bad_o] = rows, -1
    out = np.full((rows, N), -77.0, dtype)
    ob = B.shifted(out, shift) if shift else B.up(out)
    assert ds3.moe_mx_matmul(B.up(x), B.up(xs), B.up(x_rows), 1, B.up(off), B.up(w), B.up(ws), FP4, ob,
                             F16 if dtype == np.float16 else F32, B.up(out_rows), rows, rows, E, K, N) == -1
    y = R.grouped(R.decode(x, xs, FP8), R.decode(w, ws, FP4).reshape(E, N, K), off, np.where(x_rows < rows, x_rows, 0))
    y[bad_x] = 0.0
    live = np.setdiff1d(np.arange(off[-1]), [bad_o])
    out[out_rows[live]] = y[live].astype(np.float32).astype(dtype)
    assert_bitexact(B.down(ob, dtype, (rows, N)), out, "out")


def test_matmul_rows_behind_the_last_group_are_left(ds3, B):
    x, xs = exact_rows(1, 40, 128, FP8)
    w, ws = exact_rows(2, 2 * 64, 128, FP8)
    w, ws = w.reshape(2, 64, -1), ws.reshape(2, 64, -1)
    for off in ([3, 3, 20], [0, 0, 0], [5, 30, 33]):
        off = np.array(off, np.int32)
        out = np.full((40, 64), np.nan, np.float32)
        rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, off, 40, out)
        assert rc == 0
        want = out.copy()
        y = R.grouped(R.decode(x, xs, FP8), R.decode(w, ws, FP8), off, np.arange(40))
        want[off[0]:off[-1]] = y[off[0]:off[-1]].astype(np.float32)
        assert (np.isnan(got) == np.isnan(want)).all()
        assert_bitexact(np.nan_to_num(got), np.nan_to_num(want))


def test_matmul_bad_maps_and_offsets(ds3, B):
    """Named rows outside x give zero rows, output rows outside out are
    skipped, a bad offsets table is clamped; all return -1."""
    x, xs = exact_rows(1, 10, 128, FP8)
    w, ws = exact_rows(2, 2 * 64, 128, FP8)
    w, ws = w.reshape(2, 64, -1), ws.reshape(2, 64, -1)
    xd, wd = R.decode(x, xs, FP8), R.decode(w, ws, FP8)
    off = np.array([0, 20, 40], np.int32)
    src = I.rng(5).integers(0, 10, 40).astype(np.int32)
    bad = src.copy()
    bad[[2, 19, 33]] = [-1, 10, 1 << 30]
    rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, off, 40, np.full((40, 64), 5.0, np.float32), bad)
    assert rc == -1
    want = R.grouped(xd, wd, off, src)
    want[[2, 19, 33]] = 0.0
    assert_bitexact(got, want.astype(np.float32), "zero rows")
    to = np.arange(40, dtype=np.int32)
    to[[0, 25]] = [-3, 40]
    rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, off, 40, np.full((40, 64), 5.0, np.float32), src, 1, to)
    assert rc == -1
    want = R.grouped(xd, wd, off, src)
    want[[0, 25]] = 5.0
    assert_bitexact(got, want.astype(np.float32), "skipped rows")
    for table, good in (([0, 20, 99], [0, 20, 40]), ([-5, 7, 9], [0, 7, 9])):
        rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, np.array(table, np.int32), 40,
                             np.full((40, 64), 5.0, np.float32), src)
        assert rc == -1
        want = R.grouped(xd, wd, np.array(good), src)
        want[good[-1]:] = 5.0
        assert_bitexact(got, want.astype(np.float32), "clamped")
    for table in ([0, 30, 20], [40, 0, 40], [9, 8, 7]):  # decreasing: nothing is written
        rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, np.array(table, np.int32), 40,
                             np.full((40, 64), 5.0, np.float32), src)
        assert rc == -1 and (got == 5.0).all()
    # a good call after them succeeds
    rc, _ = run_matmul(ds3, B, x, xs, w, ws, FP8, off, 40, np.zeros((40, 64), np.float32), src)
    assert rc == 0


@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_matmul_ordinary_values(ds3, B, fmt):
    """Rounded sums: at most one fp32 rounding per term."""
    rows, E, K, N = 150, 3, 2048, 200
    x, xs = R.encode(I.normal(1, (rows, K)), FP8)
    w, ws = R.encode(I.normal(2, (E, N, K), 0.0, 0.02), fmt)
    off = ragged(3, rows, E, 0.0)
    rc, got = run_matmul(ds3, B, x, xs, w, ws, fmt, off, rows, np.zeros((rows, N), np.float32))
    assert rc == 0
    xd, wd = R.decode(x, xs, FP8), R.decode(w, ws, fmt)
    want = R.grouped(xd, wd, off, np.arange(rows))
    size = R.grouped(np.abs(xd), np.abs(wd), off, np.arange(rows))
    assert (np.abs(got - want) <= K * 2.0**-23 * size).all()


def test_matmul_scale_range_and_nan(ds3, B):
    """Far-apart scales, and a NaN block that reaches exactly its row or column."""
    rows, K, N = 9, 256, 70
    x, xs = exact_rows(1, rows, K, FP8, 1)
    w, ws = exact_rows(2, N, K, FP8, 1)
    w, ws = w.reshape(1, N, K), ws.reshape(1, N, -1)
    xs[:] = np.array([20, 90, 127, 140, 180, 190, 100, 60, 127], np.uint8)[:, None]
    ws[0, :, :] = np.linspace(60, 170, N).astype(np.uint8)[:, None]
    off = np.array([0, rows], np.int32)
    rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, off, rows, np.zeros((rows, N), np.float32))
    assert rc == 0
    want = R.grouped(R.decode(x, xs, FP8), R.decode(w, ws, FP8), off, np.arange(rows))
    # every term of these sums is a normal fp32 number, and no partial sum overflows
    normal = (np.abs(want) >= 2.0**-100) & (np.abs(want) < 2.0**120)
    assert normal.mean() > 0.7
    assert_bitexact(got[normal], want.astype(np.float32)[normal], "scales")
    xs[4, 3], ws[0, 11, 0] = 255, 255
    rc, got = run_matmul(ds3, B, x, xs, w, ws, FP8, off, rows, np.zeros((rows, N), np.float32))
    nan = np.zeros((rows, N), bool)
    nan[4], nan[:, 11] = True, True
    assert (np.isnan(got) == nan).all()


def test_matmul_unaligned_scales_and_offsets_past_32_bits(ds3, B):
    """Scale bytes at an odd address; and a weight tensor of more than 2^32
    bytes, read at its far end."""
    rows, K, N = 33, 512, 64
    x, xs = exact_rows(1, rows, K, FP8)
    w, ws = exact_rows(2, N, K, FP8)
    want = R.decode(x, xs, FP8) @ R.decode(w, ws, FP8).T
    off = B.up(np.array([0, rows], np.int32))
    o = B.up(np.zeros((rows, N), np.float32))
    assert ds3.moe_mx_matmul(B.up(x), B.shifted(xs, 3), None, 1, off, B.up(w), B.shifted(ws, 1), FP8, o, F32, None, rows,
                             rows, 1, K, N) == 0, ds3.last_error()
    assert_bitexact(B.down(o, np.float32, (rows, N)), want.astype(np.float32))
    E, N2 = 130, 1 << 16  # 130 x 65536 x 512 bytes = 4.06 GiB
    big, bigs = ds3.empty(E * N2 * K), ds3.empty(E * N2 * K // 32)
    B.all += [big, bigs]
    far = (E - 1) * N2 + N2 - N
    for buf, a, row in ((big, w, K), (bigs, ws, K // 32)):
        v = ds3.buffer_view(buf, far * row, a.nbytes)
        B.all.append(v)
        assert ds3.buffer_write(v, 0, a) == 0
    off = np.zeros(E + 1, np.int32)
    off[-1] = rows
    o = ds3.empty(rows * N2 * 4)
    B.all.append(o)
    assert ds3.moe_mx_matmul(B.up(x), B.up(xs), None, 1, B.up(off), big, bigs, FP8, o, F32, None, rows, rows, E, K, N2) == 0
    got = B.down(o, np.float32, (rows, N2))[:, -N:]
    assert_bitexact(got, want.astype(np.float32), "far end")


@pytest.mark.parametrize("rows,E,K,N", [(2000, 30, 640, 900), (3000, 14, 768, 2000), (6000, 12, 1024, 1500)])
def test_matmul_gathers_where_the_workspace_cannot_grow(ds3, B, rows, E, K, N):
    """A capture before any workspace exists: wide tiles gather their rows in
    the kernel. The same call outside sorts them first; both are exact."""
    ds3.shutdown()
    assert ds3.init() == 0
    x, xs = exact_rows(1, rows // 2, K, FP8)
    w, ws = exact_rows(2, E * N, K, FP8)
    off = ragged(3, rows, E, 0.1)
    src = I.rng(4).integers(0, rows // 2, rows).astype(np.int32)
    b = [B.up(v) for v in (x, xs, src, off, w, ws)]
    outs = [B.up(np.full((rows, N), np.nan, np.float32)) for _ in range(2)]
    call = lambda o: ds3.moe_mx_matmul(b[0], b[1], b[2], 1, b[3], b[4], b[5], FP8, o, F32, None, rows // 2, rows,  # noqa: E731
                                       E, K, N)
    assert ds3.graph_begin() == 0
    rc = call(outs[0])
    g = ds3.graph_end()
    assert rc == 0, ds3.last_error()
    assert ds3.graph_launch(g) == 0
    ds3.synchronize()
    assert call(outs[1]) == 0
    want = R.grouped(R.decode(x, xs, FP8), R.decode(w, ws, FP8).reshape(E, N, K), off, src).astype(np.float32)
    for o in outs:
        assert_bitexact(B.down(o, np.float32, (rows, N)), want, "out")
    # replayed again after the workspace exists
    assert ds3.buffer_write(outs[0], 0, np.zeros((rows, N), np.float32)) == 0
    assert ds3.graph_launch(g) == 0
    ds3.synchronize()
    ds3.graph_free(g)
    assert_bitexact(B.down(outs[0], np.float32, (rows, N)), want, "replayed")


# -------------------------------------------------------------------- SwiGLU
def check_act(q, s, h, slack=0.0):
    """8-bit rows against the exact h (module docstring); slack: what the sums
    before the activation may add."""
    off = 16 * 2.0**-24 * np.abs(h) + slack
    blocks = lambda v: v.reshape(*h.shape[:-1], -1, 32)  # noqa: E731
    lo = R.block_scales(blocks(np.maximum(np.abs(h) - off, 0.0)).max(-1), FP8)
    hi = R.block_scales(blocks(np.abs(h) + off).max(-1), FP8)
    assert ((s >= lo) & (s <= hi)).all(), "scales"
    unit = np.ldexp(1.0, s.astype(np.int64) - 127)[..., None]
    v, want, off = blocks(R.decode(q, s, FP8)), blocks(h), blocks(off)
    step = np.ldexp(1.0, np.maximum(np.frexp((np.abs(want) + off) / unit)[1] - 1, -6) - 3) * unit
    near = np.clip(want, -448.0 * unit, 448.0 * unit)
    assert (np.abs(v - near) <= step / 2 + off).all(), "elements"


def exact_act(xd, wd, off, src, rw=None):
    """(h, slack) of SwiGLU over decoded rows: silu' is at most 1.1, and a sum
    is off by at most K 2^-23 sum|x w|."""
    gate, up = (R.grouped(xd, w, off, src) for w in wd)
    e_gate, e_up = (xd.shape[1] * 2.0**-23 * R.grouped(np.abs(xd), np.abs(w), off, src) for w in wd)
    h, slack = R.silu(gate) * up, 1.1 * e_gate * (np.abs(up) + e_up) + np.abs(R.silu(gate)) * e_up
    return (h, slack) if rw is None else (h * rw[:, None], slack * rw[:, None])


@pytest.mark.parametrize("rows,E,K,F", [(1, 1, 32, 32), (8, 128, 2048, 96), (40, 4, 256, 64), (65, 1, 160, 160),
                                        (300, 3, 512, 128), (500, 2, 384, 32), (900, 3, 256, 224), (33, 200, 128, 768)])
@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("mapped", [False, True])
def test_swiglu(ds3, B, rows, E, K, F, fmt, mapped):
    if fmt == FP4:
        K = -(-K // 128) * 128
    used = 2
    n_x = rows if not mapped else rows // 2 + 1
    x, xs = R.encode(I.normal(1, (n_x, K)), FP8)
    w = [R.encode(I.normal(i, (E, F, K), 0.0, K**-0.5), fmt) for i in (2, 3)]
    off = ragged(4, rows, E)
    g = I.rng(5)
    x_rows = g.integers(0, n_x * used, rows).astype(np.int32) if mapped else None
    rw = g.random(n_x * used if mapped else rows).astype(np.float32) + np.float32(0.1)
    q, s = B.up(np.full((rows + 2, F), 0x33, np.uint8)), B.up(np.full((rows + 2, F // 32), 0x33, np.uint8))
    weighted = rows != 40
    assert ds3.moe_mx_swiglu(B.up(x), B.up(xs), B.up(x_rows), used, B.up(off), B.up(w[0][0]), B.up(w[0][1]),
                             B.up(w[1][0]), B.up(w[1][1]), fmt, B.up(rw) if weighted else None, q, s, n_x, rows, E, K,
                             F) == 0, ds3.last_error()
    src = x_rows // used if mapped else np.arange(rows)
    h, slack = exact_act(R.decode(x, xs, FP8), [R.decode(*p, fmt) for p in w], off, src,
                         rw[x_rows if mapped else np.arange(rows)].astype(np.float64) if weighted else None)
    got_q, got_s = B.down(q, np.uint8, (rows + 2, F)), B.down(s, np.uint8, (rows + 2, F // 32))
    assert (got_q[rows:] == 0x33).all() and (got_s[rows:] == 0x33).all()
    check_act(got_q[:rows], got_s[:rows], h, slack)


@pytest.mark.parametrize("rows,E", [(3000, 40), (3000, 14)])
@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("mapped", [False, True])
def test_swiglu_many_tiles_per_cta(ds3, B, rows, E, fmt, mapped):
    """Several tiles for every CTA at the wide token blocks: accumulators,
    column tables, exchange buffers and weights looked up ahead pass from tile
    to tile."""
    K, F, used = 256, 1504, 4
    n_x = rows // 2
    x, xs = R.encode(I.normal(1, (rows if not mapped else n_x, K)), FP8)
    w = [R.encode(I.normal(i, (E, F, K), 0.0, K**-0.5), fmt) for i in (2, 3)]
    off, g = ragged(4, rows, E, 0.1), I.rng(5)
    x_rows = g.integers(0, n_x * used, rows).astype(np.int32) if mapped else None
    rw = g.random(n_x * used if mapped else rows).astype(np.float32) + np.float32(0.1)
    q, s = B.up(np.full((rows, F), 0x33, np.uint8)), B.up(np.full((rows, F // 32), 0x33, np.uint8))
    assert ds3.moe_mx_swiglu(B.up(x), B.up(xs), B.up(x_rows), used, B.up(off), B.up(w[0][0]), B.up(w[0][1]), B.up(w[1][0]),
                             B.up(w[1][1]), fmt, B.up(rw), q, s, len(x), rows, E, K, F) == 0, ds3.last_error()
    src = x_rows // used if mapped else np.arange(rows)
    h, slack = exact_act(R.decode(x, xs, FP8), [R.decode(*p, fmt) for p in w], off, src,
                         rw[x_rows if mapped else np.arange(rows)].astype(np.float64))
    check_act(B.down(q, np.uint8, (rows, F)), B.down(s, np.uint8, (rows, F // 32)), h, slack)


@pytest.mark.parametrize("rows,E", [(3000, 40), (3000, 14)])
@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_swiglu_gathers_where_the_workspace_cannot_grow(ds3, B, rows, E, fmt):
    """A capture before any workspace exists: every width gathers its rows in
    the kernel. Outside, the same call sorts them first where the groups are
    large; both give the same codes."""
    ds3.shutdown()
    assert ds3.init() == 0
    K, F, used = 256, 736, 2
    n_x = rows // 2
    x, xs = R.encode(I.normal(1, (n_x, K)), FP8)
    w = [R.encode(I.normal(i, (E, F, K), 0.0, K**-0.5), fmt) for i in (2, 3)]
    off, g = ragged(4, rows, E, 0.1), I.rng(5)
    x_rows = g.integers(0, n_x * used, rows).astype(np.int32)
    rw = g.random(n_x * used).astype(np.float32) + np.float32(0.1)
    b = [B.up(v) for v in (x, xs, x_rows, off, *w[0], *w[1], rw)]
    outs = [(B.up(np.zeros((rows, F), np.uint8)), B.up(np.zeros((rows, F // 32), np.uint8))) for _ in range(2)]
    call = lambda o: ds3.moe_mx_swiglu(b[0], b[1], b[2], used, *b[3:8], fmt, b[8], *o, n_x, rows, E, K, F)  # noqa: E731
    assert ds3.graph_begin() == 0
    rc = call(outs[0])
    g = ds3.graph_end()
    assert rc == 0, ds3.last_error()
    for _ in range(2):
        assert ds3.graph_launch(g) == 0
    ds3.synchronize()
    ds3.graph_free(g)
    assert call(outs[1]) == 0
    got = [(B.down(q, np.uint8, (rows, F)), B.down(s, np.uint8, (rows, F // 32))) for q, s in outs]
    assert_bitexact(got[0][0], got[1][0], "gathered and sorted elements")
    assert_bitexact(got[0][1], got[1][1], "gathered and sorted scales")
    h, slack = exact_act(R.decode(x, xs, FP8), [R.decode(*p, fmt) for p in w], off, x_rows // used,
                         rw[x_rows].astype(np.float64))
    check_act(*got[0], h, slack)


def test_swiglu_bad_rows_and_large_gates(ds3, B):
    """A row id outside x gives zeros; gates far from zero saturate silu to
    0 and the identity without NaN."""
    K, F = 128, 64
    x, xs = exact_rows(1, 4, K, FP8)
    g, gs = exact_rows(2, F, K, FP8)
    u, us = exact_rows(3, F, K, FP8)
    gs[:] += 4  # gates in the thousands
    rows = np.array([0, 3, -1, 2, 4], np.int32)
    q, s = B.up(np.full((5, F), 0x33, np.uint8)), B.up(np.full((5, F // 32), 0x33, np.uint8))
    rc = ds3.moe_mx_swiglu(B.up(x), B.up(xs), B.up(rows), 1, B.up(np.array([0, 5], np.int32)), B.up(g), B.up(gs), B.up(u),
                           B.up(us), FP8, None, q, s, 4, 5, 1, K, F)
    assert rc == -1
    got_q, got_s = B.down(q, np.uint8, (5, F)), B.down(s, np.uint8, (5, 2))
    assert (got_q[[2, 4]] == 0).all() and (got_s[[2, 4]] == 0).all()
    xd, gd, ud = R.decode(x, xs, FP8), R.decode(g, gs, FP8), R.decode(u, us, FP8)
    ok = [0, 1, 3]
    gate = xd[rows[ok]] @ gd.T
    assert np.abs(gate).max() > 500
    check_act(got_q[ok], got_s[ok], R.silu(gate) * (xd[rows[ok]] @ ud.T))


def test_swiglu_gates_where_the_exponential_leaves_the_normal_range(ds3, B):
    """silu(-87.5) is 1e-36 and comes back into range with a large up product.
    The exponential there is a whole number of 2^-149: two of them are its
    2 ulp, times gate and up."""
    gates = [-80.0, -87.5, -88.0, 88.0]
    K, F, rows = 128, 32 * len(gates), 3
    one = np.zeros((rows, K))
    one[:, :2] = 1.0
    x, xs = R.encode(one, FP8)
    g = np.zeros((F, K))
    for i, v in enumerate(gates):
        big = np.sign(v) * 80.0 if abs(v) % 8 else v  # the sum of two e4m3 values
        g[32 * i:32 * i + 32, 0], g[32 * i:32 * i + 32, 1] = big, v - big
    # the two terms have to survive one scale
    gq, gs = R.encode(g, FP8)
    gd = R.decode(gq, gs, FP8)
    assert (gd == g).all()
    u = np.zeros((F, K))
    u[:, 0] = 2.0**120
    u *= np.where(np.arange(F) % 2, 1.0, -1.5)[:, None]
    uq, us = R.encode(u, FP8)
    assert (R.decode(uq, us, FP8) == u).all()
    q, s = B.up(np.zeros((rows, F), np.uint8)), B.up(np.zeros((rows, F // 32), np.uint8))
    assert ds3.moe_mx_swiglu(B.up(x), B.up(xs), None, 1, B.up(np.array([0, rows], np.int32)), B.up(gq), B.up(gs), B.up(uq),
                             B.up(us), FP8, None, q, s, rows, rows, 1, K, F) == 0, ds3.last_error()
    gate, up = one @ g.T, one @ u.T
    slack = np.where(gate < 0, 2 * 2.0**-149 * np.abs(gate * up), 0.0)
    check_act(B.down(q, np.uint8, (rows, F)), B.down(s, np.uint8, (rows, F // 32)), R.silu(gate) * up, slack)


# ------------------------------------------------------------- the whole path
class Layer:
    """One MoE FFN half on the device: norm to 8 bits, top-k, sorted rows,
    gate / up, down, combine."""

    def __init__(self, ds3, B, T, fmt, H=256, F=96, E=16, K=4, seed=50):
        self.d, self.B, self.dims = ds3, B, (T, H, F, E, K)
        self.fmt = fmt
        F = self.F = 128 if fmt == FP4 else F
        self.x, self.r, self.g = I.normal(seed, (T, H)), I.normal(seed + 1, (T, H)), I.gamma(H, seed + 2)
        self.lg = I.normal(seed + 3, (T, E), 0.0, 2.0)
        self.w = [R.encode(I.normal(seed + 4 + i, s, 0.0, s[2] ** -0.5), fmt)
                  for i, s in enumerate(((E, F, H), (E, F, H), (E, H, F)))]
        n = T * K
        z = lambda *s: B.up(np.zeros(s, np.uint8))  # noqa: E731
        self.b = dict(x=B.up(self.x), r=B.up(self.r), g=B.up(self.g), lg=B.up(self.lg), sum=z(T * H * 4), q=z(T, H),
                      s=z(T, H // 32), idx=z(n * 4), sc=z(n * 4), off=z((E + 1) * 4), ent=z(n * 4), aq=z(n, F),
                      as_=z(n, F // 32), y=z(n * H * 4), out=z(T * H * 4))
        self.wb = [(B.up(q), B.up(s)) for q, s in self.w]

    def enqueue(self):
        T, H, _, E, K = self.dims
        b, d, wb = self.b, self.d, self.wb
        assert d.add_rms_norm_mx(b["x"], b["r"], b["g"], b["sum"], None, b["q"], b["s"], H, T, 1e-6) == 0
        assert d.router_softmax_topk(b["lg"], None, b["idx"], b["sc"], T, E, K, True) == 0
        assert d.moe_expert_rows(b["idx"], b["off"], b["ent"], None, T, E, K) == 0
        assert d.moe_mx_swiglu(b["q"], b["s"], b["ent"], K, b["off"], *wb[0], *wb[1], self.fmt, None, b["aq"], b["as_"],
                               T, T * K, E, H, self.F) == 0
        assert d.moe_mx_matmul(b["aq"], b["as_"], None, 1, b["off"], *wb[2], self.fmt, b["y"], F32, b["ent"], T * K,
                               T * K, E, self.F, H) == 0
        assert d.moe_combine_residual(b["y"], None, b["sc"], b["sum"], b["out"], T, K, H) == 0

    def outputs(self):
        T, H, _, E, K = self.dims
        f = lambda k, t, s: self.B.down(self.b[k], t, s)  # noqa: E731
        return dict(sum=f("sum", np.float32, (T, H)), q=f("q", np.uint8, (T, H)), s=f("s", np.uint8, (T, H // 32)),
                    idx=f("idx", np.int32, (T, K)), sc=f("sc", np.float32, (T, K)), off=f("off", np.int32, (E + 1,)),
                    ent=f("ent", np.int32, (T * K,)), aq=f("aq", np.uint8, (T * K, self.F)),
                    as_=f("as_", np.uint8, (T * K, self.F // 32)), y=f("y", np.float32, (T * K, H)),
                    out=f("out", np.float32, (T, H)))

    def check(self, o):
        """Every stage against the 64-bit statement over the stage before it."""
        T, H, _, E, K = self.dims
        ws, wn = R.add_norm(self.x, self.r, self.g, 1e-6)
        wq, wsc = R.encode(wn.astype(np.float32), FP8)
        assert_bitexact(o["sum"], ws)
        assert_bitexact(o["q"], wq)
        assert_bitexact(o["s"], wsc)
        off, ent, _ = R.expert_rows(o["idx"], E)
        assert_bitexact(o["off"], off)
        assert_bitexact(o["ent"], ent)
        xd = R.decode(o["q"], o["s"], FP8)
        wd = [R.decode(q, s, self.fmt) for q, s in self.w]
        check_act(o["aq"], o["as_"], *exact_act(xd, wd[:2], off, ent // K))
        ad = R.decode(o["aq"], o["as_"], FP8)
        y = np.zeros((T * K, H))
        size = np.zeros((T * K, H))
        y[ent] = R.grouped(ad, wd[2], off, np.arange(T * K))
        size[ent] = R.grouped(np.abs(ad), np.abs(wd[2]), off, np.arange(T * K))
        assert (np.abs(o["y"] - y) <= self.F * 2.0**-23 * size).all()
        sc = o["sc"].astype(np.float64)[:, :, None]
        z = o["y"].astype(np.float64).reshape(T, K, H) * sc
        # K products and K + 1 sums, half a step each
        tol = (2 * K + 1) * 2.0**-24 * (np.abs(z).sum(1) + np.abs(o["sum"]))
        assert (np.abs(o["out"] - (o["sum"] + z.sum(1))) <= tol).all()


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("T", [1, 7, 130])
def test_layer_batched(ds3, B, T, fmt):
    layer = Layer(ds3, B, T, fmt)
    assert ds3.begin_batch() == 0
    layer.enqueue()
    assert ds3.end_batch() == 0, ds3.last_error()
    layer.check(layer.outputs())


@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_layer_graph_replay_on_new_inputs(ds3, B, fmt):
    """Two layers captured in one graph, replayed back to back with inputs
    changed in between (other routing, other group sizes): each replay equals
    the checked eager result bit for bit."""
    layers = [Layer(ds3, B, 96, fmt, seed=50), Layer(ds3, B, 96, fmt, seed=80)]
    for layer in layers:  # eager first: kernels set up, results to compare with
        layer.enqueue()
    assert ds3.graph_begin() == 0
    for layer in layers:
        layer.enqueue()
    g = ds3.graph_end()
    try:
        for step in range(3):
            eager = []
            for i, layer in enumerate(layers):
                layer.lg = I.normal(200 + 10 * step + i, layer.lg.shape, 0.0, 1.0 + 3 * step)
                layer.x = I.normal(300 + 10 * step + i, layer.x.shape)
                assert ds3.buffer_write(layer.b["lg"], 0, layer.lg) == 0
                assert ds3.buffer_write(layer.b["x"], 0, layer.x) == 0
                layer.enqueue()
                eager.append(layer.outputs())
                layer.check(eager[-1])
            for _ in range(3):
                assert ds3.graph_launch(g) == 0
            ds3.synchronize()
            for layer, e in zip(layers, eager):
                for k, v in layer.outputs().items():
                    assert_bitexact(v, e[k], k)
    finally:
        ds3.graph_free(g)


@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_layers_that_sort_in_one_batch_and_in_a_graph(ds3, B, fmt):
    """Groups large enough for the row sort: two layers in one batch write the
    same workspace behind one another; captured, they replay on new inputs,
    also after a larger call has outgrown the block they were captured with."""
    layers = [Layer(ds3, B, 700, fmt, seed=50), Layer(ds3, B, 700, fmt, seed=80)]
    assert ds3.begin_batch() == 0
    for layer in layers:
        layer.enqueue()
    assert ds3.end_batch() == 0, ds3.last_error()
    for layer in layers:
        layer.check(layer.outputs())
    assert ds3.graph_begin() == 0
    for layer in layers:
        layer.enqueue()
    g = ds3.graph_end()
    try:
        for step in range(3):
            if step == 2:
                Layer(ds3, B, 9000, fmt, seed=20).enqueue()
            for i, layer in enumerate(layers):
                layer.lg = I.normal(200 + 10 * step + i, layer.lg.shape, 0.0, 1.0 + 3 * step)
                layer.x = I.normal(300 + 10 * step + i, layer.x.shape)
                assert ds3.buffer_write(layer.b["lg"], 0, layer.lg) == 0
                assert ds3.buffer_write(layer.b["x"], 0, layer.x) == 0
            for _ in range(2):
                assert ds3.graph_launch(g) == 0
            ds3.synchronize()
            for layer in layers:
                layer.check(layer.outputs())
    finally:
        ds3.graph_free(g)


@pytest.mark.parametrize("T,E,K", [(37, 16, 4), (8200, 40, 8)])
def test_rows_captured_and_combined_through_the_inverse_map(ds3, B, T, E, K):
    """moe_expert_rows in a graph, at both of its forms, replayed on other ids;
    row_of takes the sorted product's rows back to their tokens in
    moe_combine_residual, as out_rows = entries does in the product."""
    H, F = 64, 32
    a, as_ = exact_rows(1, T * K, F, FP8)
    w, ws = exact_rows(2, E * H, F, FP8)
    ad, wd = R.decode(a, as_, FP8), R.decode(w, ws, FP8).reshape(E, H, F)
    n, z = T * K, lambda *s: B.up(np.zeros(s, np.int32))  # noqa: E731
    sc, res = I.rng(3).random((T, K)).astype(np.float32), I.normal(4, (T, H))
    idx, off, ent, row, y, out, y2, out2 = z(n), z(E + 1), z(n), z(n), z(n, H), z(T, H), z(n, H), z(T, H)
    b = [B.up(v) for v in (a, as_, w, ws, sc, res)]

    def enqueue():
        assert ds3.moe_expert_rows(idx, off, ent, row, T, E, K) == 0
        for dst, to, back, o in ((y, None, row, out), (y2, ent, None, out2)):
            assert ds3.moe_mx_matmul(b[0], b[1], None, 1, off, b[2], b[3], FP8, dst, F32, to, n, n, E, F, H) == 0
            assert ds3.moe_combine_residual(dst, back, b[4], b[5], o, T, K, H) == 0

    ids = [np.argsort(I.rng(7 + i).random((T, E)), 1)[:, :K].astype(np.int32) for i in range(3)]
    assert ds3.buffer_write(idx, 0, ids[0]) == 0
    enqueue()
    assert ds3.graph_begin() == 0
    enqueue()
    g = ds3.graph_end()
    try:
        for i in ids[1:]:
            assert ds3.buffer_write(idx, 0, i) == 0
            assert ds3.graph_launch(g) == 0
            ds3.synchronize()
            want = R.expert_rows(i, E)
            for got, v in zip((B.down(v, np.int32, (k,)) for v, k in ((off, E + 1), (ent, n), (row, n))), want):
                assert_bitexact(got, v)
            ys = R.grouped(ad, wd, want[0], np.arange(n)).astype(np.float32)
            assert_bitexact(B.down(y, np.float32, (n, H)), ys, "sorted rows")
            total = B.down(out, np.float32, (T, H))
            assert_bitexact(total, B.down(out2, np.float32, (T, H)), "row_of and entries")
            terms = ys[want[2]].reshape(T, K, H).astype(np.float64) * sc[:, :, None]
            # K products and K + 1 sums, half a step each
            tol = (2 * K + 1) * 2.0**-24 * (np.abs(terms).sum(1) + np.abs(res))
            assert (np.abs(total - (res + terms.sum(1))) <= tol).all()
    finally:
        ds3.graph_free(g)


@pytest.mark.parametrize("fmt", [FP8, FP4])
def test_weights_converted_expert_by_expert(ds3, B, fmt):
    """Q8_0 expert tensors to MX weights through one expert's fp32 scratch, in
    one batch, and into a product."""
    E, N, K, rows = 5, 96, 256, 40
    g = I.rng(8)
    d = g.uniform(0.001, 0.01, (E, N, K // 32, 1)).astype(np.float16)
    codes = g.integers(-127, 128, (E, N, K // 32, 32)).astype(np.int8)
    src = B.up(np.concatenate([d.view(np.uint8), codes.view(np.uint8)], -1))
    w = (d.astype(np.float32) * codes.astype(np.float32)).reshape(E, N, K)
    per = N * K // (2 if fmt == FP4 else 1)
    tmp, q, s = (B.up(np.zeros(v, np.uint8)) for v in (N * K * 4, E * per, E * N * K // 32))

    def view(b, i, n):
        B.all.append(ds3.buffer_view(b, i * n, n))
        return B.all[-1]

    assert ds3.begin_batch() == 0
    for e in range(E):
        assert ds3.dequantize_f32(view(src, e, N * K // 32 * 34), 8, N * K, tmp) == 0, ds3.last_error()
        assert ds3.mx_quantize(tmp, F32, view(q, e, per), view(s, e, N * K // 32), fmt, N, K) == 0, ds3.last_error()
    assert ds3.end_batch() == 0, ds3.last_error()
    wq, ws = R.encode(w, fmt)
    assert_bitexact(B.down(q, np.uint8, wq.shape), wq, "elements")
    assert_bitexact(B.down(s, np.uint8, ws.shape), ws, "scales")
    x, xs = R.encode(I.normal(1, (rows, K)), FP8)
    off, out = ragged(3, rows, E), B.up(np.zeros((rows, N), np.float32))
    assert ds3.moe_mx_matmul(B.up(x), B.up(xs), None, 1, B.up(off), q, s, fmt, out, F32, None, rows, rows, E, K, N) == 0
    xd, wd = R.decode(x, xs, FP8), R.decode(wq, ws, fmt)
    want, size = (R.grouped(a, b, off, np.arange(rows)) for a, b in ((xd, wd), (np.abs(xd), np.abs(wd))))
    assert (np.abs(B.down(out, np.float32, (rows, N)) - want) <= K * 2.0**-23 * size).all()


# ------------------------------------------------------------- the workspace
class Sorted:
    """A product over mapped rows that are sorted into the workspace first, with exact operands."""

    def __init__(self, ds3, B, seed, K=2048, N=32, n_x=64):
        self.d, self.B, self.K, self.N = ds3, B, K, N
        self.x, self.xs = exact_rows(seed, n_x, K, FP8)
        w, ws = exact_rows(seed + 1, N, K, FP8)
        self.wd = R.decode(w, ws, FP8)
        self.b = [B.up(v) for v in (self.x, self.xs, w, ws)]

    def call(self, out, rows, off, n):
        x, xs, w, ws = self.b
        return self.d.moe_mx_matmul(x, xs, rows, 1, off, w, ws, FP8, out, F32, None, len(self.x), n, 1, self.K, self.N)

    def want(self, rows):
        return (R.decode(self.x, self.xs, FP8) @ self.wd.T).astype(np.float32)[rows]


def free_bytes():
    import torch

    return torch.cuda.mem_get_info()[0]


def test_workspace_of_growing_batches_is_bounded(ds3, B):
    """Batches that grow step by step: what the library keeps stays within a
    small multiple of the largest, not the sum of them all."""
    ds3.shutdown()
    assert ds3.init() == 0
    s = Sorted(ds3, B, 1)
    sizes = range(16000, 40001, 500)
    rows = I.rng(3).integers(0, 64, sizes[-1]).astype(np.int32)
    rb, ob = B.up(rows), B.up(np.zeros((sizes[-1], s.N), np.float32))
    offs = [B.up(np.array([0, n], np.int32)) for n in sizes]
    assert s.call(ob, rb, offs[0], sizes[0]) == 0  # kernels loaded, a first block
    before, scratch = free_bytes(), sizes[-1] * s.K * 33 // 32
    for n, off in zip(sizes, offs):
        assert s.call(ob, rb, off, n) == 0, ds3.last_error()
    held = before - free_bytes()
    assert_bitexact(B.down(ob, np.float32, (sizes[-1], s.N)), s.want(rows), "the largest batch")
    assert held <= 2 * scratch, f"{held >> 20} MB kept for batches of at most {scratch >> 20} MB"


@pytest.mark.parametrize("capture", ["graph_begin", "the host's"])
def test_workspace_growth_between_a_capture_and_its_replay(ds3, B, capture):
    """A captured product keeps the block that it sorts into when larger calls
    outgrow it, whoever captures the module stream; the blocks that nothing
    captured go back, inside a batch too."""
    import torch

    ds3.shutdown()
    assert ds3.init() == 0
    s = Sorted(ds3, B, 5)
    n = 3000
    rows = [I.rng(7 + i).integers(0, 64, 30 * n).astype(np.int32) for i in range(3)]
    rb = [B.up(r) for r in rows]
    out, big = B.up(np.zeros((n, s.N), np.float32)), B.up(np.zeros((30 * n, s.N), np.float32))
    off = B.up(np.array([0, n], np.int32))
    assert s.call(out, rb[0], off, n) == 0
    stream = torch.cuda.ExternalStream(ds3.stream())
    if capture == "graph_begin":
        assert ds3.graph_begin() == 0
        rc = s.call(out, rb[0], off, n)
        g = ds3.graph_end()
        replay, free = lambda: ds3.graph_launch(g), lambda: ds3.graph_free(g)  # noqa: E731
    else:
        assert ds3.begin_batch() == 0
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            rc = s.call(out, rb[0], off, n)
        assert ds3.end_batch() == 0, ds3.last_error()

        def replay():
            with torch.cuda.stream(stream):
                g.replay()
            return 0

        free = g.reset
    assert rc == 0, ds3.last_error()
    try:
        for step, m in enumerate((4, 10, 30)):
            boff = B.up(np.array([0, m * n], np.int32))
            assert ds3.begin_batch() == 0
            assert s.call(big, rb[1], boff, m * n) == 0
            assert replay() == 0
            assert s.call(big, rb[2], boff, m * n) == 0
            assert ds3.end_batch() == 0, ds3.last_error()
            assert_bitexact(B.down(out, np.float32, (n, s.N)), s.want(rows[0][:n]), f"replay {step}")
            assert_bitexact(B.down(big, np.float32, (30 * n, s.N))[: m * n], s.want(rows[2][: m * n]), f"batch {step}")
            rows[0] = I.rng(40 + step).integers(0, 64, 30 * n).astype(np.int32)
            assert ds3.buffer_write(rb[0], 0, rows[0]) == 0
    finally:
        free()


def test_workspace_that_does_not_fit(ds3, B):
    """Scratch for more rows than the device holds: the call succeeds without
    it, again and again, and smaller calls still get theirs. (The one group has
    no rows, so nothing is read or written.)"""
    s = Sorted(ds3, B, 9)
    n = 1 << 27  # 258 GiB of sorted rows
    rb, ob = ds3.empty(4 * n), ds3.empty(4 * n * 1)
    B.all += [rb, ob]
    none = B.up(np.zeros(2, np.int32))
    x, xs, w, ws = s.b
    for _ in range(3):
        assert ds3.moe_mx_matmul(x, xs, rb, 1, none, w, ws, FP8, ob, F32, None, 64, n, 1, s.K, 1) == 0, ds3.last_error()
    rows = I.rng(3).integers(0, 64, 500).astype(np.int32)
    out = B.up(np.zeros((500, s.N), np.float32))
    assert s.call(out, B.up(rows), B.up(np.array([0, 500], np.int32)), 500) == 0
    assert_bitexact(B.down(out, np.float32, (500, s.N)), s.want(rows), "out")
