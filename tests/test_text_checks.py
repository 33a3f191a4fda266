"""What the text operators refuse, and where they look in a cache, on the CPU:
the _check functions on descriptors over host memory (never read), and the
index arithmetic of the kernels (paged_cache.h) in a plain C++ build."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import text_reference as ref
from conftest import ROOT


@pytest.fixture(scope="module")
def memory():
    return np.zeros(1 << 20, np.uint8)


class Maker:
    """Tensors without a context, one after the other in host memory."""

    def __init__(self, qd, memory):
        self.qd, self.base = qd, (memory.ctypes.data + 255) & ~255
        self.at, self.keep = 0, []

    def __call__(self, n, dtype=None, at=None, shift=0):
        dtype = self.qd.BF16 if dtype is None else dtype
        size = {self.qd.BF16: 2, self.qd.I8: 1, self.qd.U32: 4, self.qd.F32: 4}[dtype]
        if at is None:
            at, self.at = self.at, (self.at + n * size + 255) & ~255
        h = self.qd.lib().h3_gpu_tensor_wrap(None, self.base + at + shift, dtype, n)
        assert h
        self.keep.append(h)
        return h


def cache(qd, new, **over):
    kw = dict(k=new(4 * 8 * 2 * 128), v=new(4 * 8 * 2 * 128), table=new(6, qd.U32),
              lengths=new(2, qd.U32), starts=new(3, qd.U32), pages=4, page_size=8, table_ld=3,
              sequences=2, kv_heads=2)
    kw.update(over)
    return qd.PagedCache(**kw)


def said(fn, desc):
    text = C.create_string_buffer(256)
    ok = fn(C.byref(desc), text, 256)
    return None if ok else text.value.decode()


def rotary(qd, new, **over):
    qkv = new(5 * (4 + 2 + 2) * 128)
    kw = dict(q_out=new(5 * 512), ldq_out=512, q=qkv, ldq=1024, k=qkv, k_offset=512, ldk=1024,
              v=qkv, v_offset=768, ldv=1024, turns=new(128, qd.U32), cache=C.pointer(cache(qd, new)),
              rows=5, heads=4, kv_heads=2, head_dim=128, rotary_dim=128, layout=1,
              attention_factor=1.0, eps=1e-6)
    kw.update({k: v(kw) if callable(v) else v for k, v in over.items()})
    return qd.RotaryDesc(**kw)


def test_wrap(qd):
    L = qd.lib()
    h = L.h3_gpu_tensor_wrap(None, 4096, qd.BF16, 7)
    assert L.h3_gpu_tensor_elements(h) == 7 and L.h3_gpu_tensor_device_ptr(h) == 4096
    assert L.h3_gpu_tensor_dtype(h) == qd.BF16
    v = L.h3_gpu_tensor_view(h, 3, 4)
    assert L.h3_gpu_tensor_device_ptr(v) == 4096 + 6
    L.h3_gpu_tensor_free(v)
    L.h3_gpu_tensor_free(h)
    assert not L.h3_gpu_tensor_wrap(None, None, qd.BF16, 7)
    assert not L.h3_gpu_tensor_wrap(None, 4097, qd.BF16, 7)
    assert not L.h3_gpu_tensor_wrap(None, 4096, 9, 7)
    assert not L.h3_gpu_tensor_wrap(None, 4096, qd.F32, (1 << 64) - 1)


@pytest.mark.parametrize("over, word", [
    (dict(), None),
    (dict(rows=0), None),
    (dict(rotary_dim=24, layout=0), None),
    (dict(q_out=lambda d: d["q"], ldq_out=1024), None),  # in place
    (dict(head_dim=96), "head_dim"),
    (dict(rotary_dim=3), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"),
    (dict(rotary_dim=130), "rotary_dim"),
    (dict(layout=2), "layout"),
    (dict(attention_factor=0.0), "attention_factor"),
    (dict(attention_factor=float("nan")), "attention_factor"),
    (dict(cache=None), "positions"),
    (dict(kv_heads=1), "K/V heads"),
    (dict(v=None), "missing"),
    (dict(k_out=lambda d: d["q_out"]), "both"),
    (dict(rows=6), "too small"),
    (dict(ldq=1020), "aligned"),
    (dict(ldq=504), "stride"),
    (dict(q_offset=4), "aligned"),
    (dict(q_out=lambda d: d["q"], ldq_out=512), "overlaps"),
    (dict(q_out=lambda d: d["q"], ldq_out=1024, q_out_offset=128), "overlaps"),
    (dict(q_out=lambda d: d["turns"]), "wrong dtype"),
    (dict(norm_q=lambda d: d["q"]), "norm"),
    (dict(q_offset=(1 << 64) - 8), "too small"),
    (dict(rows=1 << 24), "2^24 rows"),
])
def test_rotary_refusals(qd, memory, over, word):
    desc = rotary(qd, Maker(qd, memory), **over)
    got = said(qd.lib().qw_gpu_rotary_check, desc)
    assert (got is None) if word is None else (got and word in got), got


def test_rotary_without_cache(qd, memory):
    new = Maker(qd, memory)
    check = qd.lib().qw_gpu_rotary_check
    kw = dict(cache=None, v=None, positions=new(5, qd.U32), k_out=new(5 * 256), ldk_out=256)
    assert said(check, rotary(qd, new, **kw)) is None
    assert "without a cache" in said(check, rotary(qd, new, **dict(kw, v=lambda d: d["q"])))
    assert "missing" in said(check, rotary(qd, new, **dict(kw, k_out=None)))
    # q alone, and both in place in the fused rows
    assert said(check, rotary(qd, new, **dict(kw, kv_heads=0, k=None, k_out=None))) is None
    both = dict(kw, q_out=lambda d: d["q"], ldq_out=1024, k_out=lambda d: d["k"], k_out_offset=512,
                ldk_out=1024)
    assert said(check, rotary(qd, new, **both)) is None
    assert "overlap" in said(check, rotary(qd, new, **dict(both, k_out_offset=0)))
    assert "overlap" in said(check, rotary(qd, new, **dict(kw, k_out=lambda d: d["q_out"])))


@pytest.mark.parametrize("over, word", [
    (dict(page_size=12), "page_size"), (dict(page_size=4), "page_size"),
    (dict(page_size=8192), "page_size"), (dict(pages=5), "too small"), (dict(pages=0), "no pages"),
    (dict(table_ld=4), "too small"), (dict(table_ld=1 << 28), "2^31"),
    (dict(sequences=3), "too small"), (dict(kv_heads=0), "no pages"), (dict(starts=None), "missing"),
    (dict(pages=1 << 31, page_size=4096, kv_heads=1024, table_ld=1), "2^32"),
    (dict(pages=(1 << 20) - 1, page_size=4096, kv_heads=1024, table_ld=1), "too small"),
])
def test_cache_refusals(qd, memory, over, word):
    new = Maker(qd, memory)
    for dims in (dict(), dict(rows=0)):
        d = attention(qd, new, cache(qd, new, **over), **dims)
        got = said(qd.lib().qw_gpu_paged_attention_check, d)
        assert got and word in got, got


def attention(qd, new, c, **over):
    kw = dict(out=new(5 * 512), ldo=512, q=new(5 * 512), ldq=512, cache=C.pointer(c), rows=5,
              heads=4, head_dim=128, scale=0.1)
    kw.update({k: v(kw) if callable(v) else v for k, v in over.items()})
    return qd.PagedAttentionDesc(**kw)


@pytest.mark.parametrize("over, word", [
    (dict(), None), (dict(rows=0), None), (dict(rows=1, ldq=0, ldo=0), None),
    (dict(head_dim=64), "head_dim"), (dict(heads=5), "heads"), (dict(heads=0), "heads"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(rows=6), "too small"), (dict(ldo=516), "too small"),
    (dict(ldq=508), "stride"), (dict(q=None), "missing"), (dict(out=lambda d: d["q"]), "overlaps"),
    (dict(cache=None), "no cache"),
    (dict(rows=1 << 31, heads=32), "2^31"),
])
def test_attention_refusals(qd, memory, over, word):
    new = Maker(qd, memory)
    got = said(qd.lib().qw_gpu_paged_attention_check, attention(qd, new, cache(qd, new), **over))
    assert (got is None) if word is None else (got and word in got), got


def test_attention_out_over_the_cache(qd, memory):
    new = Maker(qd, memory)
    c = cache(qd, new)
    got = said(qd.lib().qw_gpu_paged_attention_check, attention(qd, new, c, out=c.k))
    assert got and "overlaps" in got


@pytest.mark.parametrize("over, word", [
    (dict(), None), (dict(rows=0), None), (dict(group=32), None),
    (dict(group=16), "groups"), (dict(group=256), "groups"), (dict(k=96), "multiple"),
    (dict(k=0), "multiple"), (dict(cols=12), "multiple of 8"), (dict(cols=1 << 30), "below 2^30"), (dict(rows=6), "too small"),
    (dict(lda=120), "stride"), (dict(lda=132, rows=4), "aligned"), (dict(weight=lambda d: d["in_"]), "dtype"),
    (dict(scales=None), "missing"), (dict(out=lambda d: d["in_"]), "overlaps"),
    (dict(bias=lambda d: d["out"]), "overlaps"), (dict(ldc=20), "stride"),
    (dict(out_offset=(1 << 64) - 4), "too small"),
])
def test_linear_refusals(qd, memory, over, word):
    new = Maker(qd, memory)
    kw = dict(out=new(5 * 24), ldc=24, in_=new(5 * 128), lda=128, weight=new(24 * 64, qd.I8),
              scales=new(24 * 4), rows=5, k=128, cols=24, group=64)
    kw.update({k: v(kw) if callable(v) else v for k, v in over.items()})
    got = said(qd.lib().qw_gpu_linear_int4_check, qd.LinearInt4Desc(**kw))
    assert (got is None) if word is None else (got and word in got), got


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=128, base=1e6), dict(rotary_dim=2, base=10000.0), dict(rotary_dim=256),
    dict(rotary_dim=64, scaling="linear", factor=8.0), dict(rotary_dim=96, scaling="ntk", factor=4.0),
    dict(rotary_dim=128, base=5e5, scaling="parts", factor=8.0, original=8192.0, low=1.0, high=4.0),
    dict(rotary_dim=128, base=1e6, scaling="yarn", factor=4.0, original=32768.0, low=1.0, high=32.0),
    dict(rotary_dim=24, base=1e4, scaling="yarn", factor=16.0, original=4096.0, low=1.0, high=32.0),
])
def test_turns(qd, kw):
    """The table against the formulas: 2^-64 of a turn, and the double's own
    rounding (the power of base and the quotients: 8 of 2^-53)."""
    how = dict(plain=0, linear=1, ntk=2, parts=3, yarn=4)[kw.get("scaling", "plain")]
    args = {"original": "original_length"}
    turns, size = qd.rope_turns(**{args.get(k, k): v for k, v in kw.items() if k != "scaling"},
                                scaling=how)
    f, want = ref.frequencies(**dict(dict(base=10000.0), **{
        {"rotary_dim": "n"}.get(k, k): v for k, v in kw.items()}))
    t = (turns[:, 0].astype(np.float64) + turns[:, 1] / 2.0 ** 32) / 2.0 ** 32
    assert np.abs(t - f / (2 * np.pi)).max() <= 2.0 ** -64 + 8 * 2.0 ** -53
    assert (np.abs(t - f / (2 * np.pi)) <= 2.0 ** -64 + f * 1e-13).all()
    assert abs(size - want) <= 1e-6


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=258), dict(rotary_dim=64, base=1.0),
    dict(rotary_dim=64, base=float("nan")), dict(rotary_dim=64, scaling=5),
    dict(rotary_dim=64, scaling=1, factor=0.5), dict(rotary_dim=2, scaling=2, factor=2.0),
    dict(rotary_dim=64, scaling=3, factor=2.0, original_length=100.0, low=4.0, high=1.0),
    dict(rotary_dim=64, scaling=4, factor=2.0, original_length=0.0, low=1.0, high=32.0)])
def test_turns_refusals(qd, kw):
    with pytest.raises(ValueError):
        qd.rope_turns(**kw)


HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "kernels/paged_cache.h"
/* every index that tables of any values lead to, as the kernels take them */
int main() {
    srand(7);
    auto any = [](unsigned most) -> uint32_t {
        const int r = rand() % 8;
        const uint32_t v = ((uint32_t)rand() << 16) ^ (uint32_t)rand();
        return r == 0 ? 0xffffffffu : r == 1 ? v : r == 2 ? 0u : (uint32_t)(v % (most + 2));
    };
    long reads = 0;
    for (int round = 0; round < 4000; round++) {
        qw_cache_args c = {};
        c.pages = 1 + rand() % 9, c.page_shift = 3 + rand() % 4, c.table_ld = 1 + rand() % 7;
        c.sequences = 1 + rand() % 5, c.kv_heads = 1 + rand() % 3;
        const uint32_t rows = rand() % 40, D = 128, size = 1u << c.page_shift;
        std::vector<uint32_t> table(c.sequences * c.table_ld), len(c.sequences), st(c.sequences + 1);
        for (auto &x : table) x = any(c.pages);
        for (auto &x : len) x = any(c.table_ld * size);
        for (auto &x : st) x = any(rows);
        c.table = table.data(), c.lengths = len.data(), c.starts = st.data();
        const uint64_t all = (uint64_t)c.pages * size * c.kv_heads * D * 2; /* bytes */
        for (uint32_t s = 0; s < c.sequences; s++) {
            const qw_span sp = qw_cache_span(c, s, rows);
            if ((uint64_t)sp.begin + sp.rows > rows || sp.length > c.table_ld * size) return puts("span"), 1;
            for (uint32_t i = 0; i < sp.rows; i++) {
                const int64_t p = qw_cache_place(sp, i);
                if (p >= (int64_t)sp.length) return puts("place"), 1;
                if (p < 0) continue;
                const uint64_t e = qw_cache_entry(c, s, (uint32_t)p);
                if (e >= table.size()) return puts("entry"), 1;
                if (table[e] < c.pages)
                    for (uint32_t h = 0; h < c.kv_heads; h++)
                        if ((qw_cache_at(c, table[e], (uint32_t)p, h, D) + D) * 2 > all) return puts("store"), 1;
            }
            /* loads of 4 tokens, also past the end, as a tile rounds up */
            for (uint32_t t = 0; t < c.table_ld * size + 256; t += 4) {
                const uint64_t e = qw_cache_entry(c, s, t);
                if (e >= table.size() || e < (uint64_t)s * c.table_ld || e >= (uint64_t)(s + 1) * c.table_ld)
                    return puts("entry of a load"), 1;
                const uint32_t page = t < sp.length && table[e] < c.pages ? table[e] : 0xffffffffu;
                if (page == 0xffffffffu) continue; /* an extent of none */
                for (uint32_t h = 0; h < c.kv_heads; h++) {
                    const uint64_t at = qw_cache_at(c, page, t, h, D) * 2;
                    const uint32_t n = qw_cache_bytes(c, t, 4, sp.length, D);
                    if (!n || at + n > all) return puts("load"), 1;
                    /* the extent holds whole tokens below the end, no other */
                    for (uint32_t k = 0; k < 4; k++) {
                        const bool in = (uint64_t)k * c.kv_heads * D * 2 + D * 2 <= n;
                        if (in != (t + k < sp.length)) return puts("extent"), 1;
                        if (in != ((uint64_t)k * c.kv_heads * D * 2 < n)) return puts("part of a token"), 1;
                    }
                    reads++;
                }
            }
        }
    }
    printf("ok %ld\n", reads);
    return 0;
}
"""


def test_cache_indices_stay_in_bounds(tmp_path):
    src, exe = tmp_path / "h.cpp", tmp_path / "h"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", "-I",
                    os.path.join(ROOT, "qwen-metal_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True, timeout=120)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.startswith("ok "), out.stdout + out.stderr


def test_code_object_has_every_text_kernel(qd):
    import re
    src = open(os.path.join(ROOT, "qwen-metal_amd", "csrc", "h3_gpu_text.inc")).read()
    names = re.findall(r'"(qw_\w+)"', src[src.index("t_names[T_COUNT]"):src.index("};", src.index("t_names[T_COUNT]"))])
    blob = open(os.path.join(qd.LIB_DIR, "qwen_text_kernels.hsaco"), "rb").read()
    assert len(names) > 10
    for n in names:
        assert n.encode() in blob, n
