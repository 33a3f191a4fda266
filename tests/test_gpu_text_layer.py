"""The text operators one after another, as a model's layer runs them, on tensors
of another context, and over a cache whose offsets pass 32 bits."""
import ctypes as C

import numpy as np
import pytest

import text_reference as ref
from test_gpu_linear_int4 import weight

pytestmark = pytest.mark.gpu
SENTINEL = 0x4D21
SCALE = 1.0 / np.sqrt(128.0)


class Layer:
    """q | k | v projection, norm and rotation into the cache, attention and the
    output projection of one layer, enqueued without a wait between them."""

    def __init__(self, gpu, qd, rng, width, heads, kv, group=64):
        self.gpu, self.qd, self.heads, self.kv, self.group = gpu, qd, heads, kv, group
        self.width, self.cols = width, (heads + 2 * kv) * 128
        self.up = weight(rng, self.cols, width, group, True)
        self.down = weight(rng, width, heads * 128, group, False)
        self.bias = ref.normal(rng, self.cols, std=0.3)
        self.norms = [ref.normal(rng, 128, std=0.1, mean=1.0) for _ in range(2)]
        self.dev = [gpu.put(np.ascontiguousarray(t).view(np.int8 if i == 0 else np.uint16).ravel())
                    for w in (self.up, self.down) for i, t in enumerate(w) if t is not None]
        self.dev += [gpu.put(t) for t in (self.bias, *self.norms)]
        self.turns, _ = qd.rope_turns(128, 1e6)
        self.table = gpu.put(self.turns.ravel())

    def run(self, x, rows, cache, max_new, max_length):
        """(q | k | v, turned q, attention, out) as device tensors"""
        gpu, qd, L = self.gpu, self.qd, self.qd.lib()
        w1, s1, z1, w2, s2, bias, nq, nk = self.dev
        qkv, q, att = (gpu.new(rows * n, qd.BF16) for n in (self.cols, *[self.heads * 128] * 2))
        for t in (q, att):
            t.write(np.full(t.n, SENTINEL, np.uint16))
        out = gpu.new(rows * self.width, qd.BF16)
        up = qd.LinearInt4Desc(out=qkv.h, ldc=self.cols, in_=x.h, lda=self.width, weight=w1.h,
                               scales=s1.h, zeros=z1.h, bias=bias.h, rows=rows, k=self.width,
                               cols=self.cols, group=self.group)
        turn = qd.RotaryDesc(q_out=q.h, ldq_out=self.heads * 128, q=qkv.h, ldq=self.cols, k=qkv.h,
                             k_offset=self.heads * 128, ldk=self.cols, v=qkv.h,
                             v_offset=(self.heads + self.kv) * 128, ldv=self.cols, norm_q=nq.h,
                             norm_k=nk.h, turns=self.table.h, cache=C.pointer(cache), rows=rows,
                             heads=self.heads, kv_heads=self.kv, head_dim=128, rotary_dim=128,
                             layout=qd.ROPE_HALF, attention_factor=1.0, eps=1e-6)
        see = qd.PagedAttentionDesc(out=att.h, ldo=self.heads * 128, q=q.h, ldq=self.heads * 128,
                                    cache=C.pointer(cache), rows=rows, heads=self.heads,
                                    head_dim=128, max_new=max_new, max_length=max_length,
                                    scale=SCALE)
        down = qd.LinearInt4Desc(out=out.h, ldc=self.width, in_=att.h, lda=self.heads * 128,
                                 weight=w2.h, scales=s2.h, rows=rows, k=self.heads * 128,
                                 cols=self.width, group=self.group)
        ok = (L.qw_gpu_linear_int4(gpu.h, C.byref(up)) and
              L.qw_gpu_rotary_bf16(gpu.h, C.byref(turn)) and
              L.qw_gpu_paged_attention_bf16(gpu.h, C.byref(see)) and
              L.qw_gpu_linear_int4(gpu.h, C.byref(down)))
        gpu.check(ok, "layer")
        return qkv, q, att, out

    def check(self, b, x, got):
        """Each stage against 64 bits of what the stages before it left; b holds
        the cache as it is after the call."""
        heads, kv = self.heads, self.kv
        qkv, q, att, out = (t.read() for t in got)
        qkv = qkv.reshape(b.rows, -1)
        ref.close(qkv, *ref.linear4(x, *self.up, self.group, self.bias))
        mine = np.arange(int(b.starts[0]), int(b.starts[-1]))
        seq = np.searchsorted(b.starts, mine, "right") - 1
        place = b.lengths[seq].astype(np.int64) - (b.starts[seq + 1] - mine)
        f, _ = ref.frequencies(128, 1e6)
        split = qkv.reshape(b.rows, -1, 128)[mine]
        q = q.reshape(b.rows, heads, 128)
        ref.close(q[mine], *ref.rotary(split[:, :heads], place, f, 1.0, "half", self.norms[0]))
        page, slot = b.table[seq, place // b.page], place % b.page
        ref.close(b.k[page, slot],
                  *ref.rotary(split[:, heads:heads + kv], place, f, 1.0, "half", self.norms[1]))
        assert np.array_equal(b.v[page, slot], split[:, heads + kv:])
        att = att.reshape(b.rows, heads, 128)
        ref.close(att, *ref.attention(b, q, np.full(att.shape, SENTINEL, np.uint16), SCALE))
        ref.close(out.reshape(b.rows, -1), *ref.linear4(att.reshape(b.rows, -1), *self.down,
                                                        self.group))


def test_a_prompt_and_its_next_tokens(gpu, qd):
    """Three users: chunks of a prompt, one token each, a mix, and tokens again
    with one user gone, in one cache."""
    rng = np.random.default_rng(0)
    heads, kv, width, page = 8, 2, 256, 16
    layer = Layer(gpu, qd, rng, width, heads, kv)
    total = [60, 130, 90]
    b = ref.Batch(rng, [0, 0, 0], total, kv, page, fill=0x7FC0)
    b.k[...] = b.v[...] = 0x7FC0  # nothing in the cache yet
    ck, cv, table = (gpu.put(t.ravel()) for t in (b.k, b.v, b.table))
    have = np.zeros(3, np.int64)
    for new, pad in (([33, 100, 0], 3), ([1, 1, 70], 0), ([1, 1, 1], 5), ([2, 20, 1], 0), ([0, 1, 1], 1)):
        have += new
        b.new, b.lengths = new, have.astype(np.uint32)
        b.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        b.rows = sum(new) + pad
        x = ref.normal(rng, b.rows, width)
        meta = [gpu.put(t) for t in (b.lengths, b.starts)]
        cache = qd.PagedCache(ck.h, cv.h, table.h, meta[0].h, meta[1].h, b.pages, page, b.ld, 3, kv)
        got = layer.run(gpu.put(x.ravel()), b.rows, cache, max(new), int(have.max()))
        gpu.submit()
        b.k, b.v = (t.read().reshape(b.k.shape) for t in (ck, cv))
        layer.check(b, x, got)
    # the places of no token are as they were
    free = np.ones(b.k.shape[:2], bool)
    for s in range(3):
        _, p, slot = b.slots(s)
        free[p, slot] = False
    assert (b.k[free] == 0x7FC0).all() and (b.v[free] == 0x7FC0).all()


def test_tensors_of_another_context(gpu, qd):
    """Memory wrapped for a second context: its calls, on its own stream, read
    and write it once the first one's work is over."""
    rng = np.random.default_rng(1)
    w, s, z = weight(rng, 64, 512, 32, True)
    x = ref.normal(rng, 7, 512)
    own = [gpu.put(t) for t in (x.ravel(), w.view(np.int8).ravel(), s.ravel(), z.ravel(),
                                np.zeros(7 * 64, np.uint16))]
    gpu.submit()
    other = qd.Gpu()
    try:
        t = [other.wrap(qd.lib().h3_gpu_tensor_device_ptr(o.h), o.n, o.dtype) for o in own]
        d = qd.LinearInt4Desc(out=t[4].h, ldc=64, in_=t[0].h, lda=512, weight=t[1].h,
                              scales=t[2].h, zeros=t[3].h, rows=7, k=512, cols=64, group=32)
        other.check(qd.lib().qw_gpu_linear_int4(other.h, C.byref(d)), "linear")
        other.submit()
        for v in t:
            v.free()
    finally:
        other.close()
    ref.close(own[4].read().reshape(7, 64), *ref.linear4(x, w, s, z, 32))


@pytest.mark.parametrize("past, new", [([150, 70], [1, 1]), ([90, 200], [40, 70])])
def test_a_cache_past_32_bits(gpu, qd, past, new):
    """K and V of 9.4 GB each, the batch's pages behind element 2^32 but for a
    few at the front."""
    rng = np.random.default_rng(2)
    heads, kv, page, pages = 16, 8, 64, 72000
    size = page * kv * 128
    b = ref.Batch(rng, past, new, kv, page, spare=0, fill=0x7FC0)
    assert (pages - b.pages) * size > 1 << 32
    real = np.array([i if i < 2 else pages - 1 - i for i in range(b.pages)], np.uint32)
    big = [gpu.new(pages * size, qd.BF16) for _ in range(2)]
    try:
        for t, small in zip(big, (b.k, b.v)):
            for i in range(b.pages):
                t.view(int(real[i]) * size, size).write(small[i])
        there = b.table != ref.NONE
        table = np.where(there, real[np.where(there, b.table, 0)], ref.NONE).astype(np.uint32)
        meta = [gpu.put(t.ravel()) for t in (table, b.lengths, b.starts)]
        cache = qd.PagedCache(big[0].h, big[1].h, *(t.h for t in meta), pages, page, b.ld, 2, kv)
        layer = Layer(gpu, qd, rng, 128, heads, kv, group=32)
        x = ref.normal(rng, b.rows, 128)
        got = layer.run(gpu.put(x.ravel()), b.rows, cache, max(new), int(b.lengths.max()))
        gpu.submit()
        for t, small in zip(big, (b.k, b.v)):
            for i in range(b.pages):
                small[i] = t.view(int(real[i]) * size, size).read().reshape(small[i].shape)
        layer.check(b, x, got)
    finally:
        for t in big:
            t.free()
