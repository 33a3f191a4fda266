"""qw_gpu_rotary_bf16 against its formula in 64 bits: layouts, parts of the
head, scaled frequencies, far positions, the norm ahead of it, in place, and
into a paged cache (what is not written keeps its bits)."""
import ctypes as C

import numpy as np
import pytest

import text_reference as ref

pytestmark = pytest.mark.gpu
SENTINEL = 0x4D21


def call(gpu, qd, **kw):
    keep = [v for v in kw.values()]
    for k, v in kw.items():
        kw[k] = v.h if isinstance(v, qd.Tensor) else v
    d = qd.RotaryDesc(**kw)
    gpu.check(qd.lib().qw_gpu_rotary_bf16(gpu.h, C.byref(d)), "rotary")
    gpu.submit()
    return keep


def turns(gpu, qd, n, base=1e6, **kw):
    t, size = qd.rope_turns(n, base, **kw)
    return gpu.put(t.ravel()), size


SCALINGS = {"plain": {}, "linear": dict(factor=8.0), "ntk": dict(factor=4.0),
            "parts": dict(factor=8.0, original_length=8192.0, low=1.0, high=4.0),
            "yarn": dict(factor=4.0, original_length=32768.0, low=1.0, high=32.0)}


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim, n", [(128, 128), (128, 64), (128, 24), (128, 2), (128, 100),
                                    (64, 64), (64, 48), (256, 256), (256, 130)])
@pytest.mark.parametrize("rows, heads, kv, norm", [(1, 4, 1, True), (7, 3, 3, False),
                                                   (33, 32, 8, True)])
def test_beside(gpu, qd, layout, dim, n, rows, heads, kv, norm):
    rng = np.random.default_rng(dim * 1000 + n + rows)
    x = ref.normal(rng, rows, heads + kv, dim, std=2.0)
    w = [ref.normal(rng, dim, std=0.3, mean=1.0) for _ in range(2)] if norm else [None, None]
    pos = rng.integers(0, 5000, rows).astype(np.uint32)
    table, size = turns(gpu, qd, n)
    src = gpu.put(x.ravel())
    q, k = (gpu.put(np.full(rows * h * dim, SENTINEL, np.uint16)) for h in (heads, kv))
    kw = dict(q_out=q, ldq_out=heads * dim, k_out=k, ldk_out=kv * dim, q=src,
              ldq=(heads + kv) * dim, k=src, k_offset=heads * dim, ldk=(heads + kv) * dim,
              positions=gpu.put(pos), turns=table, rows=rows, heads=heads, kv_heads=kv,
              head_dim=dim, rotary_dim=n, layout=int(layout == "half"), attention_factor=size,
              eps=1e-6)
    if norm:
        kw.update(norm_q=gpu.put(w[0]), norm_k=gpu.put(w[1]))
    call(gpu, qd, **kw)
    f, _ = ref.frequencies(n, 1e6)
    for t, part, weight in ((q, x[:, :heads], w[0]), (k, x[:, heads:], w[1])):
        want, tol = ref.rotary(part, pos, f, 1.0, layout, weight)
        ref.close(t.read().reshape(want.shape), want, tol)
    assert np.array_equal(src.read().reshape(x.shape), x)


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_scaled_and_far(gpu, qd, scaling, layout):
    """Positions up to the last 32-bit one: the reference's angle in 64 bits is
    2^32 radians with 2^-53 of it, 5e-7 off, a tenth of the tolerance's 2e-6 of
    two values; the table's entry is 2^-65 off, 2^-33 of a turn there."""
    rng = np.random.default_rng(5)
    pos = np.array([0, 1, 2, 4095, 32767, 131071, 1000003, 16777217, 123456789, 0xFFFFFFFF],
                   np.uint32)
    rows, heads = len(pos), 2
    x = ref.normal(rng, rows, heads, 128)
    table, size = turns(gpu, qd, 128, scaling=list(SCALINGS).index(scaling), **SCALINGS[scaling])
    out = gpu.new(x.size, qd.BF16)
    call(gpu, qd, q_out=out, ldq_out=256, q=gpu.put(x.ravel()), ldq=256, positions=gpu.put(pos),
         turns=table, rows=rows, heads=heads, head_dim=128, rotary_dim=128,
         layout=int(layout == "half"), attention_factor=size)
    kw = {("original" if k == "original_length" else k): v for k, v in SCALINGS[scaling].items()}
    f, factor = ref.frequencies(128, 1e6, scaling, **kw)
    assert abs(factor - size) < 1e-6
    # angles modulo a turn from the table itself at the far end, where 64-bit
    # floating angles are too coarse: compared up to 2^24 by the formula
    near = pos <= 16777217
    want, tol = ref.rotary(x[near], pos[near], f, factor, layout)
    ref.close(out.read().reshape(x.shape)[near], want, tol)
    t = np.asarray(table.read()).reshape(-1, 2).astype(object)
    exact = [[(int(p) * (int(a) << 32 | int(b))) % 2 ** 64 / 2 ** 64 for a, b in t] for p in pos]
    angle = 2 * np.pi * np.array(exact, float)
    xs = ref.f64(x)
    a, b = (xs[..., :64], xs[..., 64:]) if layout == "half" else (xs[..., 0::2], xs[..., 1::2])
    c, s = factor * np.cos(angle)[:, None], factor * np.sin(angle)[:, None]
    y = np.concatenate([a * c - b * s, a * s + b * c], -1)
    m = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    got = out.read().reshape(x.shape)
    if layout == "interleaved":
        got = np.concatenate([got[..., 0::2], got[..., 1::2]], -1)
    ref.close(got, y, ref.HALF_STEP * np.abs(y) + 2e-6 * factor * m)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("n", [128, 40])
def test_in_place(gpu, qd, layout, n):
    """q and k of fused q | k | v rows where they are: the bits of the call
    beside, v and the rows' ends untouched."""
    rng = np.random.default_rng(n)
    rows, heads, kv = 19, 4, 2
    ld = (heads + 2 * kv) * 128 + 8
    x = ref.normal(rng, rows, ld)
    pos = gpu.put(np.arange(100, 100 + rows, dtype=np.uint32))
    table, _ = turns(gpu, qd, n)
    w = gpu.put(ref.normal(rng, 128, std=0.2, mean=1.0))
    src, fused = gpu.put(x.ravel()), gpu.put(x.ravel())
    q, k = gpu.new(rows * heads * 128, qd.BF16), gpu.new(rows * kv * 128, qd.BF16)
    kw = dict(ldq=ld, k_offset=heads * 128, ldk=ld, positions=pos, turns=table, rows=rows,
              heads=heads, kv_heads=kv, head_dim=128, rotary_dim=n, layout=layout,
              attention_factor=1.0, eps=1e-6, norm_q=w, norm_k=w)
    call(gpu, qd, q_out=q, ldq_out=heads * 128, k_out=k, ldk_out=kv * 128, q=src, k=src, **kw)
    call(gpu, qd, q_out=fused, ldq_out=ld, k_out=fused, k_out_offset=heads * 128, ldk_out=ld,
         q=fused, k=fused, **kw)
    want = x.copy()
    want[:, :heads * 128] = q.read().reshape(rows, -1)
    want[:, heads * 128:(heads + kv) * 128] = k.read().reshape(rows, -1)
    assert np.array_equal(fused.read().reshape(rows, ld), want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 64, 4096])
@pytest.mark.parametrize("past, new, front, back", [
    ([0], [1], 0, 0), ([17], [1], 0, 0), ([5, 0, 63, 200], [3, 40, 1, 0], 0, 0),
    ([0, 9, 4], [0, 0, 5], 2, 3), (list(range(70)), [1] * 70, 0, 1), ([-2, 3], [5, 4], 0, 0)])
@pytest.mark.parametrize("given", [False, True])
def test_into_the_cache(gpu, qd, dim, page, past, new, front, back, given):
    """K and V at their tokens' places, nothing else of the cache, nor of q's
    rows outside the sequences (or before a short sequence's first token)."""
    rng = np.random.default_rng(page + len(past))
    heads, kv = 6, 2
    b = ref.Batch(rng, past, new, kv, page, pad_front=front, pad_back=back, head_dim=dim,
                  holes=[(0, 0)] if len(past) == 4 else [])
    ld = (heads + 2 * kv) * dim
    x = ref.normal(rng, b.rows, heads + 2 * kv, dim)
    w = [ref.normal(rng, dim, std=0.2, mean=1.0) for _ in range(2)]
    pos = rng.integers(0, 9000, b.rows).astype(np.uint32)
    out = np.full((b.rows, heads, dim), SENTINEL, np.uint16)
    q, ck, cv, src = (gpu.put(t.ravel()) for t in (out, b.k, b.v, x))
    table, _ = turns(gpu, qd, dim // 2)
    dev = [gpu.put(t.ravel()) for t in (b.table, b.lengths, b.starts)]
    cache = qd.PagedCache(ck.h, cv.h, *(t.h for t in dev), b.pages, page, b.ld, len(new), kv)
    kw = dict(q_out=q, ldq_out=heads * dim, q=src, ldq=ld, k=src, k_offset=heads * dim, ldk=ld,
              v=src, v_offset=(heads + kv) * dim, ldv=ld, norm_q=gpu.put(w[0]),
              norm_k=gpu.put(w[1]), turns=table, cache=C.pointer(cache), rows=b.rows, heads=heads,
              kv_heads=kv, head_dim=dim, rotary_dim=dim // 2, layout=1, attention_factor=1.0,
              eps=1e-6)
    if given:
        kw["positions"] = gpu.put(pos)
    call(gpu, qd, **kw)
    f, _ = ref.frequencies(dim // 2, 1e6)
    want_q, tol_q = ref.f64(out), np.zeros(out.shape)
    want_k, tol_k, want_v = ref.f64(b.k), np.zeros(b.k.shape), b.v.copy()
    for s in range(len(new)):
        for i in range(new[s]):
            r, p = int(b.starts[s]) + i, int(b.lengths[s]) - new[s] + i
            if p < 0:
                continue
            at = pos[r:r + 1] if given else [p]
            want_q[r:r + 1], tol_q[r:r + 1] = ref.rotary(x[r:r + 1, :heads], at, f, 1.0, "half", w[0])
            pg = b.table[s, p // page]
            if pg < b.pages:
                y, t = ref.rotary(x[r:r + 1, heads:heads + kv], at, f, 1.0, "half", w[1])
                want_k[pg, p % page], tol_k[pg, p % page] = y[0], t[0]
                want_v[pg, p % page] = x[r, heads + kv:]
    ref.close(q.read().reshape(out.shape), want_q, tol_q)
    ref.close(ck.read().reshape(b.k.shape), want_k, tol_k)
    assert np.array_equal(cv.read().reshape(b.v.shape), want_v)


def test_tables_of_any_values(gpu, qd):
    """Starts, lengths and pages that make no sense: nothing outside the
    tensors is touched (guards around the outputs keep their bits), the call
    ends. What the kernel makes of the indexes is checked on the CPU."""
    rng = np.random.default_rng(3)
    heads, kv, rows, page, pages = 4, 2, 21, 8, 5
    guard = 4096
    x = gpu.put(ref.normal(rng, rows, heads + 2 * kv, 128).ravel())
    table, _ = turns(gpu, qd, 128)
    n = pages * page * kv * 128
    big = [gpu.put(np.full(m + 2 * guard, SENTINEL, np.uint16)) for m in (n, n, rows * heads * 128)]
    ck, cv, q = (t.view(guard, t.n - 2 * guard) for t in big)
    for _ in range(12):
        dev = [gpu.put(rng.choice(np.array([0, 1, 4, 5, 7, 20, 21, 22, 1 << 31, 0xFFFFFFFF],
                                           np.uint32), m)) for m in (3 * 2, 3, 4)]
        cache = qd.PagedCache(ck.h, cv.h, *(t.h for t in dev), pages, page, 2, 3, kv)
        ld = (heads + 2 * kv) * 128
        call(gpu, qd, q_out=q, ldq_out=heads * 128, q=x, ldq=ld, k=x, k_offset=heads * 128,
             ldk=ld, v=x, v_offset=(heads + kv) * 128, ldv=ld, turns=table,
             cache=C.pointer(cache), rows=rows, heads=heads, kv_heads=kv, head_dim=128,
             rotary_dim=128, layout=0, attention_factor=1.0)
    for t in big:
        v = t.read()
        assert (v[:guard] == SENTINEL).all() and (v[-guard:] == SENTINEL).all()


def test_refusals_on_the_device(gpu, qd):
    """A refused call says why and launches nothing."""
    t = gpu.put(np.zeros(1024, np.uint16))
    before = gpu.stats().direct_dispatches
    d = qd.RotaryDesc(q_out=t.h, q=t.h, rows=1, heads=1, head_dim=128, rotary_dim=128)
    assert not qd.lib().qw_gpu_rotary_bf16(gpu.h, C.byref(d))
    assert "rotary" in gpu.error()
    assert not qd.lib().qw_gpu_rotary_bf16(gpu.h, None)
    assert gpu.stats().direct_dispatches == before
