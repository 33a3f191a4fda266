"""qw_gpu_linear_int4, its quantizer and its widening, against 64 bits."""
import ctypes as C

import numpy as np
import pytest

import text_reference as ref

pytestmark = pytest.mark.gpu
SENTINEL = 0x4D21


def weight(rng, cols, k, group, zeros):
    q = rng.integers(0, 16, (cols, k)).astype(np.uint8)
    s = ref.bf16(rng.uniform(0.001, 0.02, (cols, k // group)))
    z = ref.bf16(rng.integers(0, 16, (cols, k // group))) if zeros else None
    return q[:, 0::2] | (q[:, 1::2] << 4), s, z


def linear(gpu, qd, x, w, s, z, bias, group, lda=None, ldc=None):
    rows, k = x.shape
    cols = w.shape[0]
    lda, ldc = lda or k, ldc or cols
    xs = np.full((rows, lda), 0x7FC0, np.uint16)  # NaN between the rows
    xs[:, :k] = x
    out = gpu.put(np.full(rows * ldc + 8, SENTINEL, np.uint16))
    keep = [gpu.put(xs.ravel()), gpu.put(w.view(np.int8).ravel()), gpu.put(s.ravel())]
    opt = [gpu.put(t.ravel()) if t is not None else None for t in (z, bias)]
    d = qd.LinearInt4Desc(out=out.h, out_offset=4, ldc=ldc, in_=keep[0].h, lda=lda,
                          weight=keep[1].h, scales=keep[2].h, zeros=opt[0].h if opt[0] else None,
                          bias=opt[1].h if opt[1] else None, rows=rows, k=k, cols=cols,
                          group=group)
    gpu.check(qd.lib().qw_gpu_linear_int4(gpu.h, C.byref(d)), "linear int4")
    gpu.submit()
    got = out.read()
    body = got[4:4 + rows * ldc].reshape(rows, ldc)
    assert (got[:4] == SENTINEL).all() and (got[4 + rows * ldc:] == SENTINEL).all()
    assert (body[:, cols:] == SENTINEL).all()
    return body[:, :cols]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 130])
@pytest.mark.parametrize("k, cols", [(128, 8), (1024, 24), (1664, 136), (4224, 40)])
def test_against_64_bits(gpu, qd, group, rows, k, cols):
    rng = np.random.default_rng(rows * 7 + k + group)
    w, s, z = weight(rng, cols, k, group, zeros=rows % 2 == 0)
    x = ref.normal(rng, rows, k)
    bias = ref.normal(rng, cols) if cols % 16 else None
    got = linear(gpu, qd, x, w, s, z, bias, group, lda=k + 8 * (rows % 3), ldc=cols + 4 * (rows % 2))
    ref.close(got, *ref.linear4(x, w, s, z, group, bias))


@pytest.mark.parametrize("group, k", [(32, 32), (32, 96), (32, 32 * 33), (64, 64 * 5), (64, 64 * 37)])
def test_k_that_ends_inside_a_step(gpu, qd, group, k):
    rng = np.random.default_rng(k)
    w, s, z = weight(rng, 32, k, group, True)
    x = ref.normal(rng, 5, k)
    ref.close(linear(gpu, qd, x, w, s, z, None, group), *ref.linear4(x, w, s, z, group))


@pytest.mark.parametrize("rows, k, cols", [(1, 256, 16 * 1100 + 8), (3, 512, 16 * 600 + 8),
                                           (16, 4096, 16 * 300 + 8), (5, 8320, 16 * 260 + 8)])
@pytest.mark.parametrize("group, zeros", [(32, True), (64, False), (64, True), (128, True)])
def test_more_columns_than_workgroups(gpu, qd, rows, k, cols, group, zeros):
    """Several tiles of columns for some workgroups, of which a CU holds two (x
    in 64 KB) or one."""
    rng = np.random.default_rng(rows + group)
    w, s, z = weight(rng, cols, k, group, zeros)
    x, bias = ref.normal(rng, rows, k), ref.normal(rng, cols)
    ref.close(linear(gpu, qd, x, w, s, z, bias, group), *ref.linear4(x, w, s, z, group, bias))


@pytest.mark.parametrize("rows, k", [(16, 4608), (30, 384), (60, 640), (64, 256)])
@pytest.mark.parametrize("cols", [16384 - 8, 16384 + 40, 24576 + 24, 33000])
@pytest.mark.parametrize("group, zeros", [(32, True), (64, True), (128, False)])
def test_a_round_of_workgroups(gpu, qd, rows, k, cols, group, zeros):
    """Columns about what 256 workgroups of 64, 96 and 128 have; the last tiles
    and columns drawn from the rest."""
    rng = np.random.default_rng(rows + cols)
    w, s, z = weight(rng, cols, k, group, zeros)
    x, bias = ref.normal(rng, rows, k), ref.normal(rng, cols)
    got = linear(gpu, qd, x, w, s, z, bias, group)
    at = np.r_[0:200, np.sort(rng.choice(np.arange(200, cols - 200), 300, False)), cols - 200:cols]
    ref.close(got[:, at], *ref.linear4(x, w[at], s[at], z[at] if zeros else None, group, bias[at]))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows, k", [(15, 4096), (16, 4224), (16, 4480), (4, 12288), (4, 16384), (8, 8192),
                                     (9, 8192)])
def test_x_about_what_lds_holds(gpu, qd, group, rows, k):
    """x and the scales just inside and just outside of 144 KB."""
    rng = np.random.default_rng(k + rows)
    for zeros in (False, True):
        w, s, z = weight(rng, 40, k, group, zeros)
        x = ref.normal(rng, rows, k)
        ref.close(linear(gpu, qd, x, w, s, z, None, group, lda=k + 8), *ref.linear4(x, w, s, z, group))


@pytest.mark.parametrize("rows", [1, 20, 64])
def test_every_weight_at_its_place(gpu, qd, rows):
    """Unit inputs pick single weights: (q - z) s exactly, one rounding."""
    rng = np.random.default_rng(rows)
    k, cols, group = 256, 48, 32
    w, s, z = weight(rng, cols, k, group, True)
    q = np.stack([w & 15, w >> 4], -1).reshape(cols, -1, group).astype(float)
    full = ((q - ref.f64(z)[..., None]) * ref.f64(s)[..., None]).reshape(cols, k)
    for at in range(0, k, rows):
        x = np.zeros((rows, k), np.uint16)
        n = min(rows, k - at)
        x[np.arange(n), at + np.arange(n)] = 0x3F80
        got = linear(gpu, qd, x, w, s, z, None, group)
        assert np.array_equal(got[:n], ref.bf16(full.T[at:at + n]))


def test_offset_rows_keep_their_sum(gpu, qd):
    """Inputs with a mean far above their spread: what cancels against the zero
    points is the whole sum."""
    rng = np.random.default_rng(1)
    k, cols = 4096, 64
    w, s, z = weight(rng, cols, k, 128, False)
    x = ref.normal(rng, 9, k, std=0.1, mean=30.0)
    ref.close(linear(gpu, qd, x, w, s, z, None, 128), *ref.linear4(x, w, s, z, 128))


def test_infinite_row_stays_its_own(gpu, qd):
    rng = np.random.default_rng(2)
    w, s, z = weight(rng, 24, 512, 64, False)
    x = ref.normal(rng, 18, 512)
    x[7, 100], x[17, 3] = 0x7F80, 0x7FC0
    got = ref.f64(linear(gpu, qd, x, w, s, z, None, 64))
    rest = np.delete(np.arange(18), [7, 17])
    assert not np.isfinite(got[7]).any() and not np.isfinite(got[17]).any()
    want, tol = ref.linear4(x[rest], w, s, z, 64)
    assert (np.abs(got[rest] - want) <= tol).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_and_widening(gpu, qd, group, zeros):
    """Codes by the formula (a tie of w / s falls to either side of a rounding
    of the quotient, so a code may be next to the formula's where w / s is
    within 2^-22 of a half), and within half a step of the weight."""
    rng = np.random.default_rng(group)
    rows, cols = 37, 512
    w = ref.normal(rng, rows, cols, std=0.05)
    w[3] = 0
    w[4, :group] = ref.bf16(np.full(group, 0.5))
    w[5, 7] = ref.bf16([40.0])[0]
    w[6, 9] = 0x0001
    w[6, :9] = w[6, 10:] = 0
    src = gpu.put(w.ravel())
    n = rows * cols
    q, s = gpu.new(n // 2, qd.I8), gpu.new(n // group, qd.BF16)
    z = gpu.new(n // group, qd.BF16) if zeros else None
    gpu.check(qd.lib().qw_gpu_quantize_weight_int4(gpu.h, q.h, s.h, z.h if z else None, src.h,
                                                   rows, cols, group), "quantize")
    wide = gpu.new(n, qd.BF16)
    gpu.check(qd.lib().qw_gpu_dequant_int4_bf16(gpu.h, wide.h, q.h, s.h, z.h if z else None, rows,
                                                cols, group), "dequant")
    gpu.submit()
    b = q.read().view(np.uint8).reshape(rows, -1)
    code = np.stack([b & 15, b >> 4], -1).reshape(rows, -1, group).astype(float)
    v = ref.f64(w).reshape(rows, -1, group)
    hi, lo = np.maximum(v.max(-1), 0), np.minimum(v.min(-1), 0)
    f32 = np.float32
    scale = ref.bf16((f32(hi) - f32(lo)) / f32(15) if zeros else f32(np.abs(v).max(-1)) / f32(7))
    assert np.array_equal(s.read().reshape(scale.shape), scale)
    sv = ref.f64(scale)
    safe = np.where(sv > 0, sv, 1.0)
    zero = np.where(sv > 0, np.minimum(np.rint(-lo / safe), 15), 0) if zeros else np.full(sv.shape, 8.0)
    if zeros:
        assert np.array_equal(ref.f64(z.read()).reshape(zero.shape), zero)
    exact = v / safe[..., None]
    want = np.where(sv[..., None] > 0, np.clip(np.rint(exact) + zero[..., None], 0, 15), zero[..., None])
    near = np.abs(np.abs(exact - np.floor(exact)) - 0.5) < 2.0 ** -22 * np.maximum(np.abs(exact), 1)
    assert ((code == want) | (near & (np.abs(code - want) <= 1))).all()
    back = (code - zero[..., None]) * sv[..., None]
    assert np.array_equal(wide.read().reshape(rows, cols), ref.bf16(back.reshape(rows, cols)))


def test_refusals(gpu, qd):
    t = gpu.put(np.zeros(4096, np.uint16))
    i8 = gpu.new(4096, qd.I8)
    before = gpu.stats().direct_dispatches
    L = qd.lib()
    assert not L.qw_gpu_quantize_weight_int4(gpu.h, i8.h, t.h, None, t.h, 2, 128, 128)
    assert "overlaps" in gpu.error()
    assert not L.qw_gpu_quantize_weight_int4(gpu.h, i8.h, t.h, None, t.h, 2, 100, 128)
    assert not L.qw_gpu_dequant_int4_bf16(gpu.h, t.h, i8.h, t.h, None, 2, 128, 128)
    assert not L.qw_gpu_linear_int4(gpu.h, None)
    d = qd.LinearInt4Desc(rows=1, k=128, cols=8, group=128)
    assert not L.qw_gpu_linear_int4(gpu.h, C.byref(d)) and "missing" in gpu.error()
    assert gpu.stats().direct_dispatches == before
