"""qw_gpu_paged_attention_bf16 against the formula in 64 bits: single tokens,
chunks and mixes of both, ragged lengths, pages that end inside a tile, windows,
missing pages, and caches full of NaN wherever no token lies."""
import ctypes as C

import numpy as np
import pytest

import text_reference as ref

pytestmark = pytest.mark.gpu
NAN, SENTINEL = 0x7FC0, 0x4D21
SCALE = 1.0 / np.sqrt(128.0)


def attend(gpu, qd, b, q, out, window=0, max_new=None, max_length=None, ldq=None, ldo=None,
           scale=SCALE):
    """The call's result over out's own values."""
    rows, heads, _ = q.shape
    ldq, ldo = ldq or heads * 128, ldo or heads * 128
    qs = np.full((max(rows, 1), ldq), NAN, np.uint16)
    os_ = np.full((max(rows, 1), ldo), SENTINEL, np.uint16)
    qs[:rows, :heads * 128] = q.reshape(rows, heads * 128)
    os_[:rows, :heads * 128] = out.reshape(rows, heads * 128)
    dev = [gpu.put(t.ravel()) for t in (qs, os_, b.k, b.v, b.table, b.lengths, b.starts)]
    cache = qd.PagedCache(*(t.h for t in dev[2:]), b.pages, b.page, b.ld, len(b.new), b.kv)
    d = qd.PagedAttentionDesc(
        out=dev[1].h, ldo=ldo, q=dev[0].h, ldq=ldq, cache=C.pointer(cache), rows=rows,
        heads=heads, head_dim=128, window=window,
        max_new=max(b.new) if max_new is None else max_new,
        max_length=int(b.lengths.max()) if max_length is None else max_length, scale=scale)
    gpu.check(qd.lib().qw_gpu_paged_attention_bf16(gpu.h, C.byref(d)), "paged attention")
    gpu.submit()
    got = dev[1].read().reshape(-1, ldo)
    assert (got[:, heads * 128:] == SENTINEL).all()
    return got[:rows, :heads * 128].reshape(q.shape)


def check(gpu, qd, rng, b, heads, window=0, **kw):
    q = ref.normal(rng, b.rows, heads, 128, std=1.5)
    out = np.full(q.shape, SENTINEL, np.uint16)
    got = attend(gpu, qd, b, q, out, window, **kw)
    ref.close(got, *ref.attention(b, q, out, kw.get("scale", SCALE), window))
    return q, got


@pytest.mark.parametrize("heads, kv", [(4, 4), (8, 2), (7, 1), (28, 4), (32, 1), (17, 1)])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_single_tokens(gpu, qd, heads, kv, page):
    rng = np.random.default_rng(heads + page)
    past = [0, 1, 7, 30, 31, 32, 62, 63, 64, 126, 500, 1025]
    b = ref.Batch(rng, past, [1] * len(past), kv, page, fill=NAN)
    check(gpu, qd, rng, b, heads)


@pytest.mark.parametrize("window", [1, 2, 7, 32, 33, 100, 4000])
def test_single_tokens_in_a_window(gpu, qd, window):
    rng = np.random.default_rng(window)
    past = [0, 5, 31, 32, 63, 200, 777]
    b = ref.Batch(rng, past, [1] * len(past), 2, 16, fill=NAN)
    check(gpu, qd, rng, b, 8, window)


@pytest.mark.parametrize("heads, kv", [(3, 3), (8, 2), (5, 1)])
@pytest.mark.parametrize("past, new", [
    ([0], [1]), ([0], [64]), ([0], [65]), ([0], [300]), ([130], [77]), ([1], [129]),
    ([0, 70, 3], [33, 200, 1]), ([400, 0, 0, 64], [2, 0, 256, 100])])
def test_chunks(gpu, qd, heads, kv, past, new):
    rng = np.random.default_rng(sum(past) + sum(new))
    b = ref.Batch(rng, past, new, kv, 16, pad_back=3, pad_front=1, fill=NAN)
    check(gpu, qd, rng, b, heads)


@pytest.mark.parametrize("new", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("heads", [4, 8, 12])
def test_a_few_tokens(gpu, qd, new, heads):
    """The 16- and 32-row form with blocks that end inside a token's heads."""
    rng = np.random.default_rng(new * heads)
    b = ref.Batch(rng, [0, 31, 300, 64], [new, 1, new, new - 1], 2, 8, fill=NAN)
    check(gpu, qd, rng, b, heads)


@pytest.mark.parametrize("window", [1, 20, 64, 100])
@pytest.mark.parametrize("new", [3, 150])
def test_chunks_in_a_window(gpu, qd, window, new):
    rng = np.random.default_rng(window)
    b = ref.Batch(rng, [0, 250, 90], [new, new, new // 2], 2, 32, fill=NAN)
    check(gpu, qd, rng, b, 4, window)


@pytest.mark.parametrize("new", [1, 6, 120])
@pytest.mark.parametrize("window", [0, 40])
def test_missing_pages(gpu, qd, new, window):
    """Pages given up from the front, the middle and the end (the new tokens'
    own among them): not seen, and rows that see nothing are zero."""
    rng = np.random.default_rng(new)
    b = ref.Batch(rng, [200, 64, 10], [new] * 3, 2, 8, fill=NAN,
                  holes=[(0, 0), (0, 7), (0, 8), (1, 3), (2, 0), (2, 1), (2, (9 + new) // 8)])
    check(gpu, qd, rng, b, 8, window)


def test_sequences_without_keys(gpu, qd):
    """Lengths of zero, sequences shorter than their new tokens, none at all."""
    rng = np.random.default_rng(1)
    for new in ([1, 1, 1], [40, 60, 30]):
        b = ref.Batch(rng, [-new[0], 5, -new[2] + 1], new, 2, 16, fill=NAN)
        _, got = check(gpu, qd, rng, b, 8)
        assert (got[0] == 0).all()
        b.table[:] = ref.NONE
        _, got = check(gpu, qd, rng, b, 8)
        assert (got == 0).all()


@pytest.mark.parametrize("heads, kv, past", [(8, 2, [9001]), (4, 4, [3000, 17, 8100]), (32, 1, [5000])])
@pytest.mark.parametrize("page", [8, 128])
@pytest.mark.parametrize("window", [0, 2500])
def test_long_contexts_in_pieces(gpu, qd, heads, kv, past, page, window):
    rng = np.random.default_rng(heads + page)
    b = ref.Batch(rng, past, [1] * len(past), kv, page, fill=NAN)
    q, got = check(gpu, qd, rng, b, heads, window)
    out = np.full(q.shape, SENTINEL, np.uint16)
    for _ in range(3):  # counters are as they were, and the order of arrival changes nothing
        assert np.array_equal(attend(gpu, qd, b, q, out, window), got)


@pytest.mark.parametrize("past, new", [([3000], [40]), ([1500, 600], [70, 90]), ([16000], [20]),
                                       ([50000, 3000], [9, 30])])
def test_chunks_in_pieces(gpu, qd, past, new):
    rng = np.random.default_rng(past[0])
    b = ref.Batch(rng, past, new, 2, 64, fill=NAN)
    q, got = check(gpu, qd, rng, b, 8)
    out = np.full(q.shape, SENTINEL, np.uint16)
    for _ in range(3):
        assert np.array_equal(attend(gpu, qd, b, q, out), got)


@pytest.mark.parametrize("max_new, max_length", [(1, 32), (0, 0), (1000, 1), (1, 1 << 30), (5, 700)])
def test_hints_that_are_off(gpu, qd, max_new, max_length):
    rng = np.random.default_rng(max_new)
    for past, new in (([2000, 40, 0], [1, 1, 1]), ([900, 30], [50, 3])):
        b = ref.Batch(rng, past, new, 2, 16, fill=NAN)
        check(gpu, qd, rng, b, 8, max_new=max_new, max_length=max_length)


def test_a_piece_of_many_page_ids(gpu, qd):
    """One K/V head, pages of 8 and a length hint of 1: one piece of 10000 keys,
    more page ids than are held at a time."""
    rng = np.random.default_rng(0)
    b = ref.Batch(rng, [9999], [1], 1, 8, fill=NAN, holes=[(0, 300), (0, 1100)])
    check(gpu, qd, rng, b, 4, max_length=1)


@pytest.mark.parametrize("past, new, heads", [([70], [1], 4), ([40], [3], 8), ([0], [100], 4),
                                             ([90, 0], [40, 64], 8), ([2000], [40], 4),
                                             ([16000], [20], 8)])
@pytest.mark.parametrize("window", [0, 30])
def test_infinities_that_a_row_does_not_see(gpu, qd, past, new, heads, window):
    """NaN and infinities in K and V of late and early tokens: rows that see
    them have what the formula has, the others are untouched."""
    rng = np.random.default_rng(past[0])
    b = ref.Batch(rng, past, new, 2, 16, fill=NAN)
    for s in range(len(new)):
        t, page, slot = b.slots(s)
        last = len(t) - 1
        b.v[page[last], slot[last], 0, 3] = 0x7F80
        b.v[page[last], slot[last], 0, 70] = 0xFF80
        b.v[page[last], slot[last], 1, 9] = NAN
        b.v[page[last // 2], slot[last // 2], 1, 40] = 0xFF80
        b.v[page[last // 2], slot[last // 2], 0, 3] = 0xFF80
        b.k[page[max(last - 2, 0)], slot[max(last - 2, 0)], 1, 5] = NAN if last > 2 else 0x3F80
    check(gpu, qd, rng, b, heads, window)


@pytest.mark.parametrize("past, new, heads", [([30], [1], 4), ([2000], [1], 8), ([9000], [3], 8),
                                             ([700], [40], 4), ([30, 500], [200, 90], 8),
                                             ([16000], [20], 8)])
def test_nan_in_q_and_in_stretches_of_k(gpu, qd, past, new, heads):
    """NaN wherever the formula has it: a query of NaN, and keys of NaN over
    whole tiles, where a wave or a piece sees nothing else."""
    rng = np.random.default_rng(past[0])
    b = ref.Batch(rng, past, new, 2, 16, fill=NAN)
    for s in range(len(new)):
        t, page, slot = b.slots(s)
        at = slice(len(t) // 3, len(t) // 3 + 200)
        b.k[page[at], slot[at], 1] = NAN
    q = ref.normal(rng, b.rows, heads, 128, std=1.5)
    q[b.rows // 2, 0] = NAN
    out = np.full(q.shape, SENTINEL, np.uint16)
    got = attend(gpu, qd, b, q, out)
    ref.close(got, *ref.attention(b, q, out, SCALE))
    assert np.isnan(ref.f64(got[b.rows // 2, 0])).all()
    assert np.isnan(ref.f64(got[b.rows - 1, heads - 1])).all()


@pytest.mark.parametrize("new", [1, 90])
def test_scores_of_any_size(gpu, qd, new):
    """Rows whose keys give scores far apart, all very low or all equal: the
    running maximum starts anywhere and moves."""
    rng = np.random.default_rng(new)
    b = ref.Batch(rng, [300, 100], [new, new], 2, 16, fill=NAN)
    b.k[...] = ref.bf16(ref.f64(b.k) * rng.choice([0.0, 0.1, 1.0, 3.0], b.k.shape[:2] + (1, 1)))
    check(gpu, qd, rng, b, 4)
    b.k[...] = ref.bf16(np.full(b.k.shape, -0.5))
    check(gpu, qd, rng, b, 4)
    b.k[...] = 0
    check(gpu, qd, rng, b, 4)


def test_strides(gpu, qd):
    rng = np.random.default_rng(4)
    for new in ([1, 1], [60, 90]):
        b = ref.Batch(rng, [40, 7], new, 2, 16, fill=NAN)
        check(gpu, qd, rng, b, 4, ldq=8 * 128 + 24, ldo=512 + 40)


def test_shared_pages(gpu, qd):
    """Two sequences over the same first pages."""
    rng = np.random.default_rng(6)
    b = ref.Batch(rng, [64, 64], [1, 1], 2, 16)
    b.table[1, :4] = b.table[0, :4]
    check(gpu, qd, rng, b, 4)
    b = ref.Batch(rng, [64, 64], [70, 40], 2, 16)
    b.table[1, :4] = b.table[0, :4]
    check(gpu, qd, rng, b, 4)


def test_many_sequences(gpu, qd):
    rng = np.random.default_rng(8)
    n = 150
    past = rng.integers(0, 60, n)
    b = ref.Batch(rng, past, [1] * n, 1, 8, fill=NAN)
    check(gpu, qd, rng, b, 2)
    b = ref.Batch(rng, past, list(rng.integers(0, 12, n)), 1, 8, fill=NAN)
    check(gpu, qd, rng, b, 8)


def test_tables_of_any_values(gpu, qd):
    """Starts, lengths and pages that make no sense: guards around the output
    keep their bits, the call ends (the kernel's indexes are checked on the
    CPU)."""
    rng = np.random.default_rng(3)
    heads, kv, rows, page, pages, guard = 4, 2, 21, 8, 5, 4096
    n = pages * page * kv * 128
    ck, cv, q = (gpu.put(ref.normal(rng, m)) for m in (n, n, rows * heads * 128))
    big = gpu.put(np.full(rows * heads * 128 + 2 * guard, SENTINEL, np.uint16))
    out = big.view(guard, rows * heads * 128)
    for i in range(24):
        dev = [gpu.put(rng.choice(np.array([0, 1, 4, 5, 7, 20, 21, 22, 1 << 31, 0xFFFFFFFF],
                                           np.uint32), m)) for m in (3 * 2, 3, 4)]
        cache = qd.PagedCache(ck.h, cv.h, *(t.h for t in dev), pages, page, 2, 3, kv)
        d = qd.PagedAttentionDesc(out=out.h, ldo=heads * 128, q=q.h, ldq=heads * 128,
                                  cache=C.pointer(cache), rows=rows, heads=heads, head_dim=128,
                                  max_new=[1, 8, 21][i % 3], scale=SCALE)
        gpu.check(qd.lib().qw_gpu_paged_attention_bf16(gpu.h, C.byref(d)), "paged attention")
        gpu.submit()
    v = big.read()
    assert (v[:guard] == SENTINEL).all() and (v[-guard:] == SENTINEL).all()


def test_refusals_on_the_device(gpu, qd):
    before = gpu.stats().direct_dispatches
    assert not qd.lib().qw_gpu_paged_attention_bf16(gpu.h, None)
    d = qd.PagedAttentionDesc(rows=1, heads=4, head_dim=128, scale=1.0)
    assert not qd.lib().qw_gpu_paged_attention_bf16(gpu.h, C.byref(d))
    assert "no cache" in gpu.error()
    assert gpu.stats().direct_dispatches == before
