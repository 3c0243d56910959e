"""CPU tests of the argument checks of the operators that serve a batch of requests over one prompt
(k_attention_shared_rows, k_lora_rows, k_verify_draft): refused on the host, nothing queued. The buffers are made-up
aligned addresses that are never read."""
import ctypes

import pytest

from conftest import load_package

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


def shared(kc, L, work=None, out=A, oq=None, os_=None, q=A, pk=A, pv=A, prefix_seq=64, prefix=32, k=A, v=A, starts=A,
           counts=A, heads=8, kv=2, hd=64, seq=32, batch=2, rows=3, gs=0):
    L.k_attention_shared_rows(out, oq, os_, q, pk, pv, prefix_seq, prefix, k, v, starts, counts,
                              ctypes.byref(work) if work is not None else None, heads, kv, hd, seq, batch, rows, gs)
    return rejected(L)


def made_up_work(kc, L, heads=8, kv=2, hd=64, batch=2, rows=3):
    w = kc.AttentionWork()
    L.k_attention_shared_init(ctypes.byref(w), heads, kv, hd, batch, rows, A)
    assert not L.kc_last_error()
    assert w.external == 1 and w.capacity * 4 == L.k_attention_shared_bytes(heads, kv, hd, batch, rows)
    return w


@pytest.mark.parametrize("bad", [dict(heads=9), dict(heads=0), dict(kv=0), dict(hd=0), dict(hd=257), dict(batch=-1),
                                 dict(rows=-1), dict(seq=0), dict(seq=2), dict(prefix=-1), dict(prefix=65)])
def test_shared_attention_shapes(lib, bad):
    kc, L = lib
    assert "k_attention_shared_rows: invalid shape" in shared(kc, L, made_up_work(kc, L), **bad)


@pytest.mark.parametrize("missing", ["out", "q", "pk", "pv", "k", "v", "starts"])
def test_shared_attention_missing_pointers(lib, missing):
    kc, L = lib
    assert "missing output, queries, caches or starts" in shared(kc, L, made_up_work(kc, L), **{missing: None})


def test_shared_attention_quantizer_and_work(lib):
    kc, L = lib
    w = made_up_work(kc, L)
    assert "missing output" in shared(kc, L, w, oq=A, gs=64)
    assert "group size 48 does not divide the head's 64 outputs" in shared(kc, L, w, oq=A, os_=A, gs=48)
    assert "group size 0 does not divide" in shared(kc, L, w, oq=A, os_=A)
    assert "work is missing or too small" in shared(kc, L)
    assert "work is missing or too small" in shared(kc, L, w, hd=32)
    assert "work is missing or too small" in shared(kc, L, w, rows=8)
    assert "work is missing or too small" in shared(kc, L, kc.AttentionWork())


def test_shared_attention_work_arguments(lib):
    kc, L = lib
    w = kc.AttentionWork()
    L.k_attention_shared_init(ctypes.byref(w), 8, 3, 64, 2, 3, A)
    assert rejected(L) == "k_attention_shared_init: invalid shape"
    L.k_attention_shared_init(ctypes.byref(w), 8, 2, 64, 2, 3, A + 4)
    assert "16-byte aligned" in rejected(L)
    assert L.k_attention_shared_bytes(8, 2, 64, 0, 3) == 0


def lora(L, out=A, ldo=32, base=A, ldb=32, x=A, ldx=64, index=A, table=A, count=2, kind=1, max_rank=8, n=64, d=32,
         rows=4):
    L.k_lora_rows(out, ldo, base, ldb, x, ldx, index, table, count, kind, max_rank, n, d, rows)
    return rejected(L)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(n=0), dict(d=0), dict(count=-1), dict(max_rank=0),
                                 dict(max_rank=257), dict(ldx=63), dict(ldo=31), dict(ldb=31)])
def test_lora_shapes(lib, bad):
    assert "k_lora_rows: invalid shape" in lora(lib[1], **bad)


def test_lora_type_and_pointers(lib):
    kc, L = lib
    assert lora(L, kind=3) == "k_lora_rows: invalid weight type 3"
    for missing in ("out", "x", "index", "table"):
        assert "missing output, activations, row indices or adapters" in lora(L, **{missing: None})


def verify(L, accepted=A, tokens=A, target=A, ldt=100, draft=A, ldd=100, drafted=A, counts=A, uniforms=A,
           temperature=A, vocab=100, batch=2, rows=3, work=A):
    L.k_verify_draft(accepted, tokens, target, ldt, draft, ldd, drafted, counts, uniforms, temperature, vocab, batch, rows,
                     work)
    return rejected(L)


@pytest.mark.parametrize("bad", [dict(vocab=0), dict(batch=-1), dict(rows=-1), dict(rows=65), dict(ldt=99),
                                 dict(ldd=99)])
def test_verify_shapes(lib, bad):
    assert "k_verify_draft: invalid shape" in verify(lib[1], **bad)


def test_verify_pointers_and_work(lib):
    kc, L = lib
    for missing in ("accepted", "tokens", "target", "drafted", "uniforms", "temperature", "work"):
        assert "missing outputs, logits, drafts, numbers or 16-byte aligned work" in verify(L, **{missing: None})
    assert "aligned work" in verify(L, work=A + 4)
    assert "too large" in verify(L, vocab=1 << 30, ldt=1 << 30, ldd=1 << 30, batch=1 << 20)
    assert L.k_verify_bytes(0, 1, 1) == 0 and L.k_verify_bytes(100, 1, 65) == 0


def test_python_mirror_refuses_other_layouts():
    """The mirror passes addresses only: other types, devices or strides raise before any call."""
    import torch
    kc = load_package()
    a = torch.zeros(4, 4)
    with pytest.raises(kc.KernelError, match="contiguous torch.float32 CUDA tensor"):
        kc.k_attention_shared_rows(a, None, None, a, a, a, 4, 4, a, a, a, a, kc.AttentionWork(), 1, 1, 4, 4, 1, 4, 0)
    with pytest.raises(kc.KernelError, match="as many a and b matrices"):
        kc.lora_table([a], [], [1.0])


def test_python_mirror_refuses_other_types_and_small_tables():
    """Rows with strides of their own need the right type and device all the same; a table and a work have a size."""
    import torch
    kc = load_package()
    a, i = torch.zeros(4, 4), torch.zeros(4, dtype=torch.int32)
    for x in (a, a.half()):
        with pytest.raises(kc.KernelError, match="contiguous torch.float32 CUDA tensor on the current device"):
            kc.k_lora_rows(x, 4, None, 0, x, 4, i, None, 0, kc.K_F32, 4, 4, 4, 4)
    with pytest.raises(kc.KernelError, match="CUDA tensor on the current device"):
        kc.k_verify_draft(i, i, a, 4, None, 0, i, None, a, a, 4, 1, 1, a)


@pytest.fixture
def on_cpu(monkeypatch):
    """The mirror with the CPU as its device and nothing called: what passes its checks is listed."""
    kc = load_package()
    calls = []
    monkeypatch.setattr(kc, "_device", lambda: -1)  # get_device() of a CPU tensor
    monkeypatch.setattr(kc, "_call", lambda name, *args: calls.append(name))
    return kc, calls


@pytest.mark.parametrize("dtype,kind", [("float32", 0), ("bfloat16", 1), ("float16", 2)])
def test_python_mirror_holds_a_table_to_its_call(on_cpu, dtype, kind):
    """A table's adapters have a type and sizes; a call with others would read past their matrices."""
    import torch
    kc, calls = on_cpu
    t = getattr(torch, dtype)
    table = kc.lora_table([torch.zeros(8, 64, dtype=t)] * 2, [torch.zeros(32, 8, dtype=t)] * 2, [1.0, 2.0])
    x, out, index = torch.zeros(4, 128), torch.zeros(4, 64), torch.zeros(4, dtype=torch.int32)
    call = lambda kind=kind, n=64, d=32: kc.k_lora_rows(out, 64, None, 0, x, 128, index, table, 2, kind, 8, n, d, 4)  # noqa: E731
    call()
    assert calls == ["k_lora_rows"]
    for other in ((kind + 1) % 3, (kind + 2) % 3):
        with pytest.raises(kc.KernelError, match=f"table of adapters of type {kind}, 64 to 32, .* type {other}, 64 to 32"):
            call(kind=other)
    for sizes in (dict(n=128), dict(n=63), dict(d=64), dict(d=33)):
        with pytest.raises(kc.KernelError, match="for a call with"):
            call(**sizes)
    assert calls == ["k_lora_rows"]
    call(d=31)  # the first outputs alone
    assert len(calls) == 2
    with pytest.raises(kc.KernelError, match="float32, bfloat16 or float16"):
        kc.lora_table([torch.zeros(8, 64, dtype=torch.float64)], [torch.zeros(32, 8, dtype=torch.float64)], [1.0])


def test_python_mirror_refuses_columns_apart(on_cpu):
    """Rows may lie apart, a row's elements may not: transposed and sliced activations, outputs and logits."""
    import torch
    kc, calls = on_cpu
    table = kc.lora_table([torch.zeros(8, 16)], [torch.zeros(16, 8)], [1.0])
    index, good = torch.zeros(16, dtype=torch.int32), torch.zeros(16, 40)
    kc.k_lora_rows(good[:, :16], 40, good[:, 16:32], 40, good[:, 20:36], 40, index, table, 1, kc.K_F32, 8, 16, 16, 16)
    kc.k_lora_rows(good[:, :1], 40, None, 0, good[:1, :16], 40, index, table, 1, kc.K_F32, 8, 16, 16, 1)
    assert len(calls) == 2
    for bad in (good[:, :16].t(), good[:, ::2]):
        for at in range(3):
            out, base, x = [bad if i == at else good for i in range(3)]
            with pytest.raises(kc.KernelError, match="contiguous torch.float32"):
                kc.k_lora_rows(out, 40, base, 40, x, 40, index, table, 1, kc.K_F32, 8, 16, 16, 16)
    i, u, t, work = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 2), torch.ones(1), torch.zeros(1 << 16)
    for target, draft in ((good.t(), None), (good, good.t())):
        with pytest.raises(kc.KernelError, match="contiguous torch.float32"):
            kc.k_verify_draft(i[:, :1], i, target, 40, draft, 40, i[:, :1], None, u, t, 16, 1, 1, work)
    assert len(calls) == 2


def test_python_mirror_refuses_memory_elsewhere(on_cpu):
    """Works and tables on another device (here: one that holds nothing)."""
    import torch
    kc, calls = on_cpu
    a, i = torch.zeros(4, 4), torch.zeros(4, dtype=torch.int32)

    class Elsewhere:
        device = "cuda:1"
        get_device = staticmethod(lambda: 1)
        numel, element_size = staticmethod(lambda: 1 << 20), staticmethod(lambda: 1)

    with pytest.raises(kc.KernelError, match="the adapters' table must be on the current CUDA device, is on cuda:1"):
        kc.k_lora_rows(a, 4, None, 0, a, 4, i, Elsewhere(), 1, kc.K_F32, 4, 4, 4, 4)
    with pytest.raises(kc.KernelError, match="the work must be on the current CUDA device"):
        kc.k_verify_draft(i[:1], i, a, 4, None, 0, i, None, a, a, 4, 1, 1, Elsewhere())
    work = kc.AttentionWork()
    work._memory = Elsewhere()
    with pytest.raises(kc.KernelError, match="the attention work must be on the current CUDA device"):
        kc.k_attention_shared_rows(a, None, None, a, a, a, 4, 4, a, a, i, i, work, 1, 1, 4, 4, 1, 4, 0)
    assert not calls


@pytest.mark.parametrize("bad", [dict(prefix_seq=2 ** 31 - 1, prefix=2 ** 31 - 1), dict(seq=2 ** 31 - 1),
                                 dict(prefix_seq=2 ** 31 - 64, prefix=2 ** 31 - 64)])
def test_shared_attention_positions_past_the_integers(lib, bad):
    """Positions are numbered in tiles past the last one: lengths at the end of the integers would wrap."""
    kc, L = lib
    assert "k_attention_shared_rows: invalid shape" in shared(kc, L, made_up_work(kc, L), **bad)


@pytest.mark.parametrize("heads,batch,rows", [(4, 2 ** 31 - 1, 2 ** 31 - 1), (8, 2 ** 30, 2 ** 31 - 1),
                                              (2 ** 31 - 1, 2 ** 31 - 1, 4), (2 ** 16, 2 ** 24, 2 ** 24)])
def test_shared_attention_products_of_sizes_that_wrap(lib, heads, batch, rows):
    kc, L = lib
    assert L.k_attention_shared_bytes(heads, 1, 64, batch, rows) == 0
    w = kc.AttentionWork()
    L.k_attention_shared_init(ctypes.byref(w), heads, 1, 64, batch, rows, A)
    assert rejected(L) == "k_attention_shared_init: invalid shape"


@pytest.mark.parametrize("bad", [dict(n=2 ** 31 - 1, ldx=2 ** 31), dict(d=2 ** 31 - 1, ldo=2 ** 31, ldb=2 ** 31),
                                 dict(n=2 ** 31 - 8192, ldx=2 ** 31)])
def test_lora_columns_past_the_integers(lib, bad):
    """Columns are numbered in slices and steps past the last one."""
    assert "k_lora_rows: invalid shape" in lora(lib[1], **bad)
