"""CPU tests of the argument checks of the operators that serve from a paged cache (k_rope_kv_store_paged,
k_attention_paged_rows, k_token_logprobs): refused on the host, nothing queued. The buffers are made-up aligned addresses
that are never read."""
import ctypes
import subprocess

import pytest

from conftest import ROOT, load_package

A = 0x10000


@pytest.fixture(scope="module")
def lib():
    kc = load_package()
    L = kc.load()
    L.kc_set_fail_mode(kc.KC_FAIL_RETURN)
    return kc, L


def rejected(L):
    msg = L.kc_last_error()
    L.kc_clear_error()
    assert msg, "the call was accepted"
    return msg.decode()


def made_up_cache(kc, key=A, value=A, table=A, page_stride=2 * 16 * 64, kind=1, pages=9, page_size=16, max_pages=4):
    return kc.PagedCache(key, value, table, page_stride, kind, pages, page_size, max_pages)


def made_up_work(kc, heads=8, hd=64, workers=6):
    """As k_attention_paged_init leaves one (it queues its tickets' zeroing, so it needs a device)."""
    L = kc.load()
    size = L.k_attention_paged_bytes(heads, 2, hd, workers, 1)
    return kc.AttentionWork(A, -1, heads, hd, workers, 1, size // 4)


def store(kc, L, cache=None, q_out=A, q_out_ld=512, q=A, q_ld=512, k=A, v=A, kv_ld=128, rope=A, seq=64, starts=A, counts=A,
          heads=8, kv=2, hd=64, batch=2, rows=3):
    L.k_rope_kv_store_paged(q_out, q_out_ld, q, q_ld, k, v, kv_ld, ctypes.byref(cache) if cache is not None else None, rope,
                            seq, starts, counts, heads, kv, hd, batch, rows)
    return rejected(L)


def attention(kc, L, cache=None, work=None, out=A, oq=None, os_=None, q=A, starts=A, counts=A, heads=8, kv=2, hd=64,
              batch=2, rows=3, gs=0):
    L.k_attention_paged_rows(out, oq, os_, q, ctypes.byref(cache) if cache is not None else None, starts, counts,
                             ctypes.byref(work) if work is not None else None, heads, kv, hd, batch, rows, gs)
    return rejected(L)


def logprobs(L, lp=A, entropy=A, top_tokens=A, top_lp=A, logits=A, ld=100, tokens=A, vocab=100, rows=4, top=5):
    L.k_token_logprobs(lp, entropy, top_tokens, top_lp, logits, ld, tokens, vocab, rows, top)
    return rejected(L)


@pytest.mark.parametrize("bad", [dict(heads=0), dict(kv=0), dict(hd=0), dict(hd=63), dict(batch=-1), dict(rows=-1),
                                 dict(seq=0), dict(q_ld=511), dict(q_out_ld=511), dict(kv_ld=127),
                                 dict(batch=1 << 20, rows=1 << 12), dict(heads=1 << 26, q_ld=1 << 40, q_out_ld=1 << 40)])
def test_store_shapes(lib, bad):
    kc, L = lib
    assert "k_rope_kv_store_paged: invalid shape" in store(kc, L, made_up_cache(kc), **bad)


@pytest.mark.parametrize("missing", ["q_out", "q", "k", "v", "rope", "starts"])
def test_store_missing_pointers(lib, missing):
    kc, L = lib
    assert "missing queries, keys, values, rotation table or starts" in store(kc, L, made_up_cache(kc), **{missing: None})


def test_store_in_place_strides(lib):
    kc, L = lib
    assert "need one row stride" in store(kc, L, made_up_cache(kc), q_ld=512, q_out_ld=768)


CACHES = [(dict(key=None), "missing keys, values or page table"), (dict(value=None), "missing keys, values or page table"),
          (dict(table=None), "missing keys, values or page table"), (dict(kind=3), "invalid cache type"),
          (dict(kind=-1), "invalid cache type"), (dict(pages=0), "invalid pages"), (dict(page_size=0), "invalid pages"),
          (dict(max_pages=0), "invalid pages"), (dict(pages=-1), "invalid pages"),
          (dict(page_size=1 << 16, max_pages=1 << 15, page_stride=1 << 40), "invalid pages"),
          (dict(page_stride=2 * 16 * 64 - 1), "invalid page stride"), (dict(page_stride=0), "invalid page stride"),
          (dict(page_stride=(1 << 64) - 1), "invalid page stride")]


@pytest.mark.parametrize("bad,message", CACHES, ids=lambda x: str(x))
def test_caches(lib, bad, message):
    kc, L = lib
    cache = made_up_cache(kc, **bad)
    assert f"k_rope_kv_store_paged: {message}" in store(kc, L, cache)
    assert f"k_attention_paged_rows: {message}" in attention(kc, L, cache, made_up_work(kc))


def test_no_cache(lib):
    kc, L = lib
    assert "missing keys" in store(kc, L)
    assert "missing keys" in attention(kc, L, None, made_up_work(kc))


@pytest.mark.parametrize("bad", [dict(heads=9), dict(heads=0), dict(kv=0), dict(hd=0), dict(hd=257), dict(batch=-1),
                                 dict(rows=-1), dict(batch=1 << 13, rows=1 << 12)])
def test_attention_shapes(lib, bad):
    kc, L = lib
    assert "k_attention_paged_rows: invalid shape" in attention(kc, L, made_up_cache(kc), made_up_work(kc), **bad)


@pytest.mark.parametrize("missing", ["out", "q", "starts"])
def test_attention_missing_pointers(lib, missing):
    kc, L = lib
    assert "missing output, queries or starts" in attention(kc, L, made_up_cache(kc), made_up_work(kc), **{missing: None})


def test_attention_quantizer_and_work(lib):
    kc, L = lib
    c, w = made_up_cache(kc), made_up_work(kc)
    assert "missing output" in attention(kc, L, c, w, oq=A, gs=64)
    assert "group size 48 does not divide the head's 64 outputs" in attention(kc, L, c, w, oq=A, os_=A, gs=48)
    assert "group size 0 does not divide" in attention(kc, L, c, w, oq=A, os_=A)
    for other in (None, kc.AttentionWork(), made_up_work(kc, hd=32), made_up_work(kc, heads=16), made_up_work(kc, workers=5)):
        assert "work is missing or too small" in attention(kc, L, c, other)
    shared = kc.AttentionWork()
    L.k_attention_shared_init(ctypes.byref(shared), 8, 2, 64, 2, 3, A)
    assert "work is missing or too small" in attention(kc, L, c, shared)
    # and the paged work passes for no other
    L.k_attention_shared_rows(A, None, None, A, A, A, 64, 32, A, A, A, A, ctypes.byref(w), 8, 2, 64, 32, 2, 3, 0)
    assert "work is missing or too small" in rejected(L)


def test_attention_work_arguments(lib):
    kc, L = lib
    w = kc.AttentionWork()
    L.k_attention_paged_init(ctypes.byref(w), 8, 3, 64, 2, 3, A)
    assert rejected(L) == "k_attention_paged_init: invalid shape"
    L.k_attention_paged_init(ctypes.byref(w), 8, 2, 64, 2, 3, A + 4)
    assert "16-byte aligned" in rejected(L)
    assert L.k_attention_paged_bytes(8, 2, 64, 0, 3) == 0
    # any split of as many rows over requests fits one work
    assert L.k_attention_paged_bytes(8, 2, 64, 6, 1) == L.k_attention_paged_bytes(8, 2, 64, 2, 3)


@pytest.mark.parametrize("bad", [dict(vocab=0), dict(rows=-1), dict(top=-1), dict(top=33), dict(top=101), dict(ld=99),
                                 dict(vocab=4, top=5)])
def test_logprobs_shapes(lib, bad):
    assert "k_token_logprobs: invalid shape" in logprobs(lib[1], **bad)


@pytest.mark.parametrize("missing", [("logits",), ("lp",), ("tokens",), ("top_tokens",), ("top_lp",)])
def test_logprobs_pointers(lib, missing):
    assert "missing logits, log probabilities or tokens, or room" in logprobs(lib[1], **{m: None for m in missing})


def test_nothing_to_do_is_accepted(lib):
    kc, L = lib
    L.k_rope_kv_store_paged(A, 512, A, 512, A, A, 128, None, A, 64, A, A, 8, 2, 64, 0, 3)
    L.k_attention_paged_rows(A, None, None, A, None, A, A, None, 8, 2, 64, 2, 0, 0)
    L.k_token_logprobs(A, A, None, None, A, 100, A, 100, 0, 0)
    assert not L.kc_last_error()


def test_c_header_layout_matches(tmp_path):
    """PagedCache has the same layout in the C header and the Python mirror."""
    kc = load_package()
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "kernels_cuda.h"\n'
                   'int main(void) { printf("%zu %zu %zu %zu %zu\\n", sizeof(PagedCache), offsetof(PagedCache, table), '
                   'offsetof(PagedCache, page_stride), offsetof(PagedCache, type), offsetof(PagedCache, max_pages)); '
                   'return 0; }\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    P = kc.PagedCache
    assert got == [ctypes.sizeof(P), P.table.offset, P.page_stride.offset, P.type.offset, P.max_pages.offset]
