"""GPU tests of the operators that serve from a paged cache, against plain 64-bit forms of their definitions.

Tolerances, from the number of roundings (fp32: half a step is u = 2^-24 of the value):
  - storing: bitwise; the rotation is two products and a sum, each rounded, and a 16-bit value is rounded once.
  - attention: roundings taken as random, as for attention over a shared prefix: a score is a chain of head_dim roundings
    of values up to the largest score S, about sqrt(head_dim) u S off; a score off by e moves a weight by e of itself, and
    weights, sums and joins add a few u. Four standard deviations: 4 u (sqrt(head_dim) S + 8) of the largest output.
  - log probabilities: with d = M - x and means over p, a weight e^-d is off by (d + 4) u of itself (the difference or its
    product with log2 e rounded, the exponential's own 4 u), so log S by (E d + 4) u; sums in fp32 parts add 8 u. With the
    result's own rounding: u (|log p| + E d + 12). The entropy log S + T / S, T = sum e^-d d: u (H + E d^2 + 5 E d + 12 (1 +
    E d)), every term of T being off by (d + 5) u of itself and its sum by 8 u.
"""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
name_of = lambda t: str(t)[6:]  # noqa: E731


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def dev(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


class Pages:
    """A pool of pages in any order, NaN all over, and a table that names pages only for `positions[b]` positions of
    request b; the rest of the table is no page."""

    def __init__(self, kc, seed, positions, kv, page, hd, dtype, width=None, spare=3, pool=None):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in positions]
        self.page, self.hd, self.kv = page, hd, kv
        self.width = width or max(1, max(need))
        order = rng.permutation(sum(need) + spare)
        self.table = np.full((len(positions), self.width), -1, np.int32)
        self.table[:] = rng.choice([-1, 1 << 30, -(1 << 31)], self.table.shape)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (len(order), kv, page, hd)
        if pool is None:
            self.key, self.value = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        else:
            self.key, self.value = pool(shape, dtype)
        self.device_table = torch.tensor(self.table, device="cuda")
        self.cache = kc.paged_cache(self.key, self.value, self.device_table)

    def fill(self, b, keys, values):
        """Positions 0 .. of request b: keys, values [kv][n][hd]."""
        n = keys.shape[1]
        for p in range(0, n, self.page):
            m = min(self.page, n - p)
            at = int(self.table[b, p // self.page])
            self.key[at, :, :m] = keys[:, p:p + m].to(self.key.dtype)
            self.value[at, :, :m] = values[:, p:p + m].to(self.key.dtype)

    def take(self, b, n):
        """Positions [0, n) of request b, [kv][n][hd] in 64 bits."""
        ids = torch.tensor(self.table[b, :-(-n // self.page)].astype(np.int64), device="cuda")
        return tuple(x[ids].transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (self.key, self.value))


# ---- storing -----------------------------------------------------------------------------------------------------------

def rope_table(n, hd):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    cos, sin = angle.cos().float(), angle.sin().float()
    return torch.cat([torch.stack([cos, cos], -1).flatten(1), torch.stack([-sin, sin], -1).flatten(1)], 1).cuda()


def rotate(x, row, hd):
    """One row [n * hd] in fp32, product by product."""
    a, b = x.view(-1, hd // 2, 2).unbind(-1)
    c, s = row[0:hd:2], row[hd + 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).view(-1, hd)


STORE = [  # heads, kv, hd, batch, rows, page, row padding
    (1, 1, 2, 1, 1, 1, 0),
    (8, 2, 64, 1, 1, 16, 0),
    (32, 8, 128, 5, 1, 16, 0),
    (32, 8, 128, 3, 7, 24, 0),
    (14, 2, 64, 4, 33, 17, 4),
    (6, 3, 10, 3, 5, 7, 3),
    (4, 4, 34, 2, 9, 5, 1),
    (28, 4, 128, 9, 2, 64, 8),
    (8, 1, 256, 2, 130, 128, 0),
    (2, 2, 6, 3, 4, 3, 2),
]


def store_inputs(kc, case, dtype, seed=0):
    heads, kv, hd, B, R, page, pad = case
    g, rng = generator(seed + heads), np.random.default_rng(seed + R)
    counts = [int(c) for c in rng.integers(0, R + 1, B)]
    counts[-1] = R
    starts = [int(s) for s in rng.integers(0, 50, B)]
    pages = Pages(kc, seed, [s + c for s, c in zip(starts, counts)], kv, page, hd, dtype)
    q, k, v = (normal(g, B, R, n * hd + pad) for n in (heads, kv, kv))
    return pages, q, k, v, starts, counts


def stored(pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out, skip=()):
    """What the call leaves: (q_out, key, value)."""
    q_out, key, value = q_out.clone(), pages.key.clone(), pages.value.clone()
    for b in range(q.shape[0]):
        for r in range(counts[b]):
            p = starts[b] + r
            at = int(pages.table[b, p // pages.page])
            if b in skip or (b, r) in skip:
                continue
            q_out[b, r, :heads * hd] = rotate(q[b, r, :heads * hd], rope[p], hd).flatten()
            key[at, :, p % pages.page] = rotate(k[b, r, :kv * hd], rope[p], hd).to(key.dtype)
            value[at, :, p % pages.page] = v[b, r, :kv * hd].view(kv, hd).to(key.dtype)
    return q_out, key, value


def run_store(kc, pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out):
    kc.k_rope_kv_store_paged(q_out, q_out.stride(1), q, q.stride(1), k, v, k.stride(1), pages.cache, rope, rope.shape[0],
                             dev(starts), dev(counts), heads, kv, hd, q.shape[0], q.shape[1])
    return kc.status()


def same(got, want):
    bits = {4: torch.int32, 2: torch.int16}[got.element_size()]
    return torch.equal(got.view(bits), want.view(bits)) if got.is_contiguous() else same(got.contiguous(), want.contiguous())


def check_store(got, want):
    for x, y in zip(got, want):
        assert same(torch.nan_to_num(x, nan=123.0), torch.nan_to_num(y, nan=123.0))


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("case", STORE, ids=lambda c: "-".join(map(str, c)))
def test_store(kc, case, dtype):
    heads, kv, hd, B, R, page, pad = case
    pages, q, k, v, starts, counts = store_inputs(kc, case, dtype)
    rope = rope_table(50 + R, hd)
    q_out = torch.full((B, R, heads * hd + 2 * pad), -7.0, device="cuda")
    want = stored(pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out)
    assert run_store(kc, pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out) == 0
    check_store((q_out, pages.key, pages.value), want)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_store_in_place_of_one_product(kc, dtype):
    """q, k and v side by side in the rows of one product; the queries stay where they are."""
    heads, kv, hd, B, R = 8, 2, 64, 3, 4
    pages, _, _, _, starts, counts = store_inputs(kc, (heads, kv, hd, B, R, 16, 0), dtype)
    rope = rope_table(64, hd)
    qkv = normal(generator(3), B, R, (heads + 2 * kv) * hd)
    q, k, v = qkv.split([heads * hd, kv * hd, kv * hd], -1)
    before = qkv.clone()
    want = stored(pages, q, k, v, rope, starts, counts, heads, kv, hd, q)
    assert run_store(kc, pages, q, k, v, rope, starts, counts, heads, kv, hd, q) == 0
    check_store((q, pages.key, pages.value), want)
    assert torch.equal(qkv[..., heads * hd:], before[..., heads * hd:])


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_store_alignment(kc, dtype, offset):
    """Every buffer at an address of its element only, pages a stride apart that no 16 bytes divide."""
    heads, kv, hd, B, R, page = 8, 2, 64, 3, 5, 16
    shifted = lambda x: torch.cat([torch.zeros(offset, device="cuda"), x.flatten()])[offset:].view(x.shape)  # noqa: E731

    def pool(shape, dtype):
        each = shape[1] * shape[2] * shape[3] + offset
        return tuple(torch.full((shape[0] * each + offset,), float("nan"), dtype=dtype, device="cuda")[offset:]
                     .as_strided(shape, (each, shape[2] * shape[3], shape[3], 1)) for _ in range(2))

    counts, starts = [5, 0, 3], [30, 0, 2]
    pages = Pages(kc, 1, [35, 0, 5], kv, page, hd, dtype, pool=pool)
    g = generator(offset)
    q, k, v = (shifted(normal(g, B, R, n * hd)) for n in (heads, kv, kv))
    rope = shifted(rope_table(64, hd))
    q_out = shifted(torch.full((B, R, heads * hd), -7.0, device="cuda"))
    want = stored(pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out)
    assert run_store(kc, pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out) == 0
    check_store((q_out, pages.key, pages.value), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name_of)
def test_store_rounds_to_nearest(kc, dtype):
    """Ties, values beyond the type's range, its smallest ones, infinities and NaN, as torch rounds them."""
    hd, n = 64, 6
    eps = torch.finfo(dtype).eps
    special = torch.tensor([1 + eps / 2, 1 + 1.5 * eps, -1 - eps / 2, 65504.0, 65519.9, 65520.0, 1e30, 3.4e38, -3.4e38,
                            float("inf"), float("-inf"), 0.0, -0.0, 6e-8, 2.9e-8, 1e-40, 6.1e-5, 1e-45])
    v = torch.zeros(1, n, hd)
    v.view(-1)[:special.numel()] = special
    v = v.cuda()
    pages = Pages(kc, 0, [n], 1, 4, hd, dtype)
    q = torch.zeros(1, n, hd, device="cuda")
    rope = torch.zeros(n, 2 * hd, device="cuda")
    rope[:, :hd] = 1.0  # the angle 0: a pair (a, b) becomes (a - 0, 0 + b)
    assert run_store(kc, pages, q, v, v, rope, [0], [n], 1, 1, hd, torch.zeros_like(q)) == 0
    got_v = torch.cat([pages.value[int(p), 0] for p in pages.table[0]])[:n]
    assert same(got_v, v[0].to(dtype))
    got_k = torch.cat([pages.key[int(p), 0] for p in pages.table[0]])[:n]
    want_k = rotate(v[0].flatten(), rope[0], hd).to(dtype)
    assert same(torch.nan_to_num(got_k, nan=5.0), torch.nan_to_num(want_k, nan=5.0))


def test_store_is_the_contiguous_caches(kc):
    """The same rows through k_rope_kv_store_rows."""
    heads, kv, hd, R, seq = 8, 2, 128, 37, 80
    g = generator(4)
    q, k, v = (normal(g, 1, R, n * hd) for n in (heads, kv, kv))
    rope = rope_table(seq, hd)
    kc_, vc_ = (torch.zeros(kv, seq, hd, device="cuda") for _ in range(2))
    q2 = q.clone()
    kc.k_rope_kv_store_rows(q2, heads * hd, k, v, kv * hd, kc_, vc_, rope, None, 11, R, heads, kv, hd, seq)
    pages = Pages(kc, 2, [11 + R], kv, 16, hd, torch.float32)
    q_out = torch.empty_like(q)
    assert run_store(kc, pages, q, k, v, rope, [11], None, heads, kv, hd, q_out) == 0
    keys, values = pages.take(0, 11 + R)
    assert same(q_out, q2) and torch.equal(keys[:, 11:], kc_[:, 11:11 + R].double())
    assert torch.equal(values[:, 11:], vc_[:, 11:11 + R].double())


@pytest.mark.parametrize("starts,counts,rope", [([0, -1, 0], [2, 2, 2], 64), ([0, 31, 0], [2, 2, 2], 64),
                                                ([0, 2, 0], [2, 5, 2], 64), ([0, 2, 0], [2, -1, 2], 64),
                                                ([0, 2 ** 31 - 1, 0], [2, 2, 2], 64), ([0, 19, 0], [2, 2, 2], 20)])
def test_store_reports_bad_requests(kc, starts, counts, rope):
    """Only the request concerned is left out."""
    heads, kv, hd, R = 4, 2, 64, 4
    pages = Pages(kc, 3, [32, 32, 32], kv, 16, hd, torch.float16)
    g = generator(5)
    q, k, v = (normal(g, 3, R, n * hd) for n in (heads, kv, kv))
    table = rope_table(rope, hd)
    q_out = torch.full_like(q, -7.0)
    want = stored(pages, q, k, v, table, starts, [c if b != 1 else 0 for b, c in enumerate(counts)], heads, kv, hd, q_out)
    with pytest.raises(kc.KernelError):
        run_store(kc, pages, q, k, v, table, starts, counts, heads, kv, hd, q_out)
    check_store((q_out, pages.key, pages.value), want)


@pytest.mark.parametrize("page", [-1, 9, 1 << 30])
def test_store_reports_bad_pages(kc, page):
    heads, kv, hd, R = 4, 2, 64, 20
    pages = Pages(kc, 3, [32, 32, 32], kv, 16, hd, torch.bfloat16)
    pages.table[1, 1] = page
    pages.device_table[1, 1] = page
    g = generator(5)
    q, k, v = (normal(g, 3, R, n * hd) for n in (heads, kv, kv))
    rope, starts, counts = rope_table(64, hd), [0, 3, 12], [20, 20, 20]
    q_out = torch.full_like(q, -7.0)
    bad = [(1, r) for r in range(13, 20)]
    want = stored(pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out, skip=bad)
    with pytest.raises(kc.KernelError):
        run_store(kc, pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out)
    check_store((q_out, pages.key, pages.value), want)


def test_store_offsets_past_32_bits(kc):
    """A pool of more than 2^32 bytes and more than 2^31 elements: the last page is written, and nothing else."""
    kv, hd, page, heads, n_pages = 8, 128, 64, 8, 33000
    key, value = (torch.zeros(n_pages, kv, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert key.numel() > 2 ** 31
    table = dev([[n_pages - 1]])
    cache = kc.paged_cache(key, value, table)
    g = generator(1)
    q, k, v = (normal(g, 1, 2, n * hd) for n in (heads, kv, kv))
    rope = rope_table(64, hd)
    out = torch.empty_like(q)
    kc.k_rope_kv_store_paged(out, heads * hd, q, heads * hd, k, v, kv * hd, cache, rope, 64, dev([62]), None, heads, kv, hd,
                             1, 2)
    assert kc.status() == 0
    for r in range(2):
        assert same(key[-1, :, 62 + r], rotate(k[0, r], rope[62 + r], hd).bfloat16())
        assert same(value[-1, :, 62 + r], v[0, r].view(kv, hd).bfloat16())
    assert not key[:-1].any() and not value[:-1].any() and not key[-1, :, :62].any()


# ---- attention ---------------------------------------------------------------------------------------------------------

def attention_64(pages, q, starts, counts, heads, kv, hd, before):
    out, top = before.double().clone(), 1.0
    for b in range(q.shape[0]):
        if not counts[b]:
            continue
        keys, values = pages.take(b, starts[b] + counts[b])
        for r in range(counts[b]):
            n = starts[b] + r + 1
            s = torch.einsum("kgd,kpd->kgp", q[b, r].double().view(kv, heads // kv, hd), keys[:, :n]) / hd ** 0.5
            top = max(top, float(s.abs().max()))
            out[b, r] = torch.einsum("kgp,kpd->kgd", s.softmax(-1), values[:, :n]).reshape(-1)
    return out, top


def run_attention(kc, pages, q, starts, counts, heads, kv, hd, gs=0, work=None, out=None):
    B, R = q.shape[:2]
    out = torch.full_like(q, -7.0) if out is None else out
    oq = torch.full(q.shape, 99, dtype=torch.int8, device="cuda") if gs else None
    os_ = torch.full((B, R, heads * hd // gs), -1.0, device="cuda") if gs else None
    work = work or kc.paged_attention_work(heads, kv, hd, B, R)
    kc.k_attention_paged_rows(out, oq, os_, q, pages.cache, dev(starts), dev(counts), work, heads, kv, hd, B, R, gs)
    kc.status()
    return (out, oq, os_) if gs else out


def close(got, want, hd, top):
    tol = 4 * U * (hd ** 0.5 * top + 8) * max(float(want.abs().max()), 1e-30)
    assert float((got.double() - want).abs().max()) <= tol


def fill_normal(pages, g, lengths, scale_k=1.0, scale_v=1.0):
    for b, n in enumerate(lengths):
        if n:
            pages.fill(b, normal(g, pages.kv, n, pages.hd) * scale_k, normal(g, pages.kv, n, pages.hd) * scale_v)


ATTENTION = [  # heads, kv, hd, batch, rows, longest, page
    (1, 1, 64, 1, 1, 1, 1),
    (1, 1, 128, 1, 1, 2, 16),
    (8, 2, 64, 1, 1, 128, 16),
    (8, 2, 128, 2, 3, 70, 16),
    (32, 8, 128, 5, 4, 133, 17),
    (32, 8, 64, 3, 2, 1000, 24),
    (32, 8, 128, 1, 1, 5000, 64),
    (32, 8, 64, 40, 5, 257, 9),
    (16, 16, 64, 9, 1, 200, 8),
    (14, 2, 64, 7, 8, 450, 32),
    (28, 4, 128, 6, 7, 520, 128),
    (8, 2, 32, 11, 3, 203, 5),
    (6, 2, 48, 3, 2, 78, 16),
    (12, 3, 96, 4, 3, 150, 16),
    (4, 1, 256, 2, 2, 71, 3),
    (6, 3, 10, 3, 4, 46, 7),
    (2, 1, 33, 2, 2, 40, 1),
    (48, 1, 128, 2, 3, 400, 16),
    (48, 1, 64, 3, 13, 300, 64),
    (4, 4, 128, 70, 1, 300, 256),
    (32, 8, 128, 2, 130, 400, 16),
    (8, 8, 64, 1, 77, 100, 8),
    (16, 2, 32, 2, 33, 90, 12),
    (20, 4, 80, 3, 2, 333, 16),
    (5, 1, 256, 4, 6, 150, 16),
]


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(map(str, c)))
def test_attention(kc, case, dtype):
    heads, kv, hd, B, R, S, page = case
    g, rng = generator(heads * 1000 + S), np.random.default_rng(S + B)
    counts = [int(c) for c in rng.integers(0, min(R, S) + 1, B)]
    counts[-1] = min(R, S)
    starts = [int(rng.integers(0, S - c + 1)) for c in counts]
    starts[-1] = S - counts[-1]
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    # What no row sees is NaN: the rest of a last page, other pages, the rows out of use; unused requests have no pages.
    pages = Pages(kc, S, lengths, kv, page, hd, dtype)
    fill_normal(pages, g, lengths)
    q = 1.5 * normal(g, B, R, heads * hd)
    for b in range(B):
        q[b, counts[b]:] = float("nan")
    got = run_attention(kc, pages, q, starts, counts, heads, kv, hd)
    want, top = attention_64(pages, q, starts, counts, heads, kv, hd, torch.full_like(q, -7.0))
    for b in range(B):
        assert (got[b, counts[b]:] == -7.0).all()
    close(got, want, hd, top)


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("heads,kv,hd,R", [(8, 2, 128, 1), (8, 2, 64, 3), (6, 3, 48, 2)])
def test_attention_strides_and_alignment(kc, heads, kv, hd, R, dtype, offset):
    """Queries, outputs and caches at addresses of their elements only, pages an odd stride apart, in any combination that the
    kernels tell apart."""
    B, page, lengths = 3, 16, [70, 200, 5]
    shifted = lambda x, by: torch.cat([torch.zeros(by, device="cuda"), x.flatten()])[by:].view(x.shape)  # noqa: E731
    for base, gap in ((offset, 0), (0, offset), (offset, offset)):
        def pool(shape, dtype):
            each = shape[1] * shape[2] * shape[3] + gap
            return tuple(torch.full((shape[0] * each + base,), float("nan"), dtype=dtype, device="cuda")[base:]
                         .as_strided(shape, (each, shape[2] * shape[3], shape[3], 1)) for _ in range(2))

        pages = Pages(kc, 1, lengths, kv, page, hd, dtype, pool=pool)
        g = generator(offset)
        fill_normal(pages, g, lengths)
        q = shifted(normal(g, B, R, heads * hd), offset % 4)
        out = shifted(torch.full((B, R, heads * hd), -7.0, device="cuda"), base % 4)
        starts = [n - R for n in lengths]
        run_attention(kc, pages, q, starts, [R] * B, heads, kv, hd, out=out)
        want, top = attention_64(pages, q, starts, [R] * B, heads, kv, hd, q)
        close(out, want, hd, top)


def test_attention_all_rows_without_counts(kc):
    heads, kv, hd, B, R = 8, 2, 128, 3, 2
    pages = Pages(kc, 1, [70, 2, 33], kv, 16, hd, torch.bfloat16)
    g = generator(2)
    fill_normal(pages, g, [70, 2, 33])
    q = normal(g, B, R, heads * hd)
    got = run_attention(kc, pages, q, [68, 0, 31], None, heads, kv, hd)
    want, top = attention_64(pages, q, [68, 0, 31], [2, 2, 2], heads, kv, hd, q)
    close(got, want, hd, top)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_attention_peaked_and_rising_scores(kc, dtype):
    """Scores that rise along the positions (the running maximum moves all the time) or fall, and single winners."""
    heads, kv, hd, n = 4, 1, 128, 700
    q = torch.ones(3, 1, heads * hd, device="cuda")
    pages = Pages(kc, 5, [n] * 3, kv, 16, hd, dtype)
    rise = torch.linspace(-40, 40, n, device="cuda")[None, :, None] / hd ** 0.5
    values = normal(generator(6), kv, n, hd)
    pages.fill(0, rise.expand(kv, n, hd), values)
    pages.fill(1, -rise.expand(kv, n, hd), values)
    one = torch.zeros(kv, n, hd, device="cuda")
    one[:, 333] = 60 / hd ** 0.5
    pages.fill(2, one, values)
    starts, counts = [n - 1] * 3, [1] * 3
    got = run_attention(kc, pages, q, starts, counts, heads, kv, hd)
    want, top = attention_64(pages, q, starts, counts, heads, kv, hd, q)
    close(got, want, hd, top)


@pytest.mark.parametrize("hd", [128, 64, 96, 33])
@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("wrong", [float("nan"), float("inf"), float("-inf"), "largest"])
def test_attention_keeps_to_what_a_row_sees(kc, hd, dtype, wrong):
    """A later draft's key and value of any kind reach the rows from it on, and no others."""
    heads, kv, R = 8, 2, 4
    wrong = torch.finfo(dtype).max if wrong == "largest" else wrong
    g = generator(hd)
    for n, bad in itertools.product([R, 64 + R, 130], [1, 3]):
        pages = Pages(kc, n, [n], kv, 16, hd, dtype)
        fill_normal(pages, g, [n])
        at = n - R + bad
        place = int(pages.table[0, at // 16]), slice(None), at % 16
        pages.key[place], pages.value[place] = 0.0, 0.0
        q = normal(g, 1, R, heads * hd)
        want, top = attention_64(pages, q, [n - R], [R], heads, kv, hd, q)
        pages.key[place], pages.value[place] = wrong, wrong
        got = run_attention(kc, pages, q, [n - R], [R], heads, kv, hd)
        close(got[:, :bad], want[:, :bad], hd, top)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e-30), (torch.bfloat16, 1e-6), (torch.bfloat16, 1e8),
                                        (torch.bfloat16, 1e30), (torch.float16, 1e-4), (torch.float16, 60.0),
                                        (torch.float16, 3000.0), (torch.float32, 1e-30), (torch.float32, 1e30)], ids=str)
def test_attention_of_any_power(kc, hd, dtype, size):
    """Small and large keys and values over the type's range; queries are scaled the other way."""
    heads, kv, lengths = 8, 2, [300, 1]
    pages = Pages(kc, 5, lengths, kv, 16, hd, dtype)
    g = generator(7)
    fill_normal(pages, g, lengths, size, size)
    q = normal(g, 2, 1, heads * hd) / size
    got = run_attention(kc, pages, q, [299, 0], [1, 1], heads, kv, hd)
    want, top = attention_64(pages, q, [299, 0], [1, 1], heads, kv, hd, q)
    close(got, want, hd, top)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name_of)
def test_attention_large_values_of_no_weight(kc, hd, dtype):
    """A value of the type's largest size whose weight is far below a rounding takes no bits of the others."""
    heads, kv, n = 4, 1, 200
    pages = Pages(kc, 5, [n], kv, 16, hd, dtype)
    g = generator(8)
    keys, values = 0.01 * normal(g, kv, n, hd), normal(g, kv, n, hd)
    drop = 150.0 if dtype == torch.bfloat16 else 60.0  # e^-150 of 3.4e38 and e^-60 of 65504: nothing beside 1
    q = torch.ones(1, 1, heads * hd, device="cuda")
    keys[:, ::7] = -drop / hd ** 0.5
    values[:, ::7] = torch.finfo(dtype).max
    pages.fill(0, keys, values)
    got = run_attention(kc, pages, q, [n - 1], [1], heads, kv, hd)
    want, _ = attention_64(pages, q, [n - 1], [1], heads, kv, hd, q)
    live = keys.double()[:, [i for i in range(n) if i % 7]]
    close(got, want, hd, float(live.sum(-1).abs().max()) / hd ** 0.5 + 1)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_attention_of_the_largest_values(kc, dtype):
    """The mean of many values of the type's largest size is finite, and it."""
    heads, kv, hd, n = 8, 2, 128, 1500
    pages = Pages(kc, 5, [n], kv, 64, hd, dtype)
    most = torch.finfo(dtype).max
    keys = normal(generator(1), kv, n, hd)
    pages.fill(0, keys, torch.full((kv, n, hd), most, device="cuda"))
    q = 0.1 * normal(generator(2), 1, 1, heads * hd)
    got = run_attention(kc, pages, q, [n - 1], [1], heads, kv, hd)
    # a mean of equal values: weights and their sum are rounded alike in number and sum, 64 positions or so to a chain
    assert torch.isfinite(got).all()
    assert float((got.double() / most - 1).abs().max()) <= 4 * U * (8 + 8)


def norm_error(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("case", [(32, 8, 128, 1, 1, 8192), (32, 8, 64, 4, 1, 4099), (32, 8, 128, 8, 5, 2500),
                                  (28, 4, 128, 3, 1, 3001)], ids=lambda c: "-".join(map(str, c)))
def test_attention_error(kc, case, dtype):
    """The root mean square error: scores sqrt(head_dim) roundings of their size or fewer, weights and sums a few."""
    heads, kv, hd, B, R, n = case
    pages = Pages(kc, 9, [n] * B, kv, 32, hd, dtype)
    g = generator(9)
    fill_normal(pages, g, [n] * B)
    q = 1.5 * normal(g, B, R, heads * hd)
    got = run_attention(kc, pages, q, [n - R] * B, [R] * B, heads, kv, hd)
    want, top = attention_64(pages, q, [n - R] * B, [R] * B, heads, kv, hd, q)
    # a score's size is 1.5 in the root mean square; a weight that counts has one of up to about 5
    assert norm_error(got, want) <= U * (hd ** 0.5 * 1.5 + 8)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("hd,gs", [(128, 64), (64, 64), (64, 16), (128, 128), (96, 32)])
def test_attention_quantizes_its_output(kc, hd, gs, dtype):
    heads, kv, B, R = 8, 2, 5, 3
    lengths = [100, 3, 400, 0, 65]
    pages = Pages(kc, 3, lengths, kv, 16, hd, dtype)
    g = generator(3)
    fill_normal(pages, g, lengths)
    q = normal(g, B, R, heads * hd)
    counts = [3, 3, 1, 0, 2]
    starts = [n - c for n, c in zip(lengths, counts)]
    out, oq, os_ = run_attention(kc, pages, q, starts, counts, heads, kv, hd, gs)
    plain = run_attention(kc, pages, q, starts, counts, heads, kv, hd)
    assert same(out, plain)
    for b in range(B):
        c = counts[b]
        assert (oq[b, c:] == 99).all() and (os_[b, c:] == -1).all() and (out[b, c:] == -7).all()
        if c:
            wq, ws = torch.empty_like(oq[b, :c]), torch.empty_like(os_[b, :c])
            kc.k_quantize_rows(wq, ws, out[b, :c].contiguous(), heads * hd, c, heads * hd, gs)
            assert torch.equal(oq[b, :c], wq) and same(os_[b, :c], ws)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("starts,counts", [([80, -1, 80], [1, 1, 1]), ([80, 96, 80], [1, 1, 1]), ([80, 95, 80], [1, 2, 1]),
                                           ([80, 5, 80], [1, 4, 1]), ([80, 5, 80], [1, -3, 1]),
                                           ([80, 2 ** 31 - 1, 80], [1, 1, 1])])
def test_attention_reports_bad_requests(kc, starts, counts, dtype):
    heads, kv, hd, R = 4, 2, 64, 3
    pages = Pages(kc, 3, [96, 96, 96], kv, 16, hd, dtype)
    g = generator(3)
    fill_normal(pages, g, [96] * 3)
    q = normal(g, 3, R, heads * hd)
    out = torch.full_like(q, -7.0)
    with pytest.raises(kc.KernelError):
        run_attention(kc, pages, q, starts, counts, heads, kv, hd, out=out)
    good = [c if b != 1 else 0 for b, c in enumerate(counts)]
    want, top = attention_64(pages, q, starts, good, heads, kv, hd, torch.full_like(q, -7.0))
    close(out, want, hd, top)
    assert (out[1] == -7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("hd", [128, 64, 48])
@pytest.mark.parametrize("page,index", [(-1, 0), (1 << 30, 4), (-(1 << 31), 40), (10 ** 6, 62)])
def test_attention_reports_bad_pages(kc, page, index, hd, dtype):
    """A page that is none, wherever it lies among a request's, leaves that request's rows alone as they were."""
    heads, kv, R, n = 8, 2, 2, 1000
    pages = Pages(kc, 3, [n] * 3, kv, 16, hd, dtype)
    g = generator(3)
    fill_normal(pages, g, [n] * 3)
    pages.device_table[1, index] = page
    q = normal(g, 3, R, heads * hd)
    out = torch.full_like(q, -7.0)
    with pytest.raises(kc.KernelError):
        run_attention(kc, pages, q, [n - R] * 3, [R] * 3, heads, kv, hd, out=out)
    assert (out[1] == -7).all()
    want, top = attention_64(pages, q, [n - R] * 3, [R, 0, R], heads, kv, hd, torch.full_like(q, -7.0))
    close(out, want, hd, top)
    # the work is as good as new
    pages.device_table[1, index] = int(pages.table[1, index])
    got = run_attention(kc, pages, q, [n - R] * 3, [R] * 3, heads, kv, hd)
    want, top = attention_64(pages, q, [n - R] * 3, [R] * 3, heads, kv, hd, q)
    close(got, want, hd, top)


def test_attention_shared_pages(kc):
    """Requests whose first pages are one prompt's, and one request of drafts against the same rows as requests."""
    heads, kv, hd, page = 8, 2, 128, 16
    pages = Pages(kc, 3, [100, 100], kv, page, hd, torch.bfloat16)
    g = generator(3)
    fill_normal(pages, g, [100, 100])
    pages.table[1, :3] = pages.table[0, :3]
    pages.device_table.copy_(torch.tensor(pages.table))
    q = normal(g, 2, 1, heads * hd)
    got = run_attention(kc, pages, q, [99, 60], [1, 1], heads, kv, hd)
    want, top = attention_64(pages, q, [99, 60], [1, 1], heads, kv, hd, q)
    close(got, want, hd, top)
    pages.device_table[1] = pages.device_table[0]
    pages.table[1] = pages.table[0]
    apart = run_attention(kc, pages, q, [98, 99], [1, 1], heads, kv, hd)
    as_drafts = run_attention(kc, pages, q.view(1, 2, -1), [98], [2], heads, kv, hd)
    want, top = attention_64(pages, q, [98, 99], [1, 1], heads, kv, hd, q)
    close(apart, want, hd, top)
    close(as_drafts.view(2, 1, -1), want, hd, top)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("batch,rows,heads,kv,hd,page", [(1500, 1, 8, 8, 64, 16), (700, 3, 16, 8, 64, 8), (2100, 1, 4, 1, 128, 32)])
def test_attention_many_requests(kc, batch, rows, heads, kv, hd, page, dtype):
    """More requests than threads, short and of very different lengths."""
    rng = np.random.default_rng(batch)
    counts = [int(c) for c in rng.integers(0, rows + 1, batch)]
    lengths = [c + int(rng.integers(0, 3) * rng.integers(0, 90)) if c else 0 for c in counts]
    lengths[7] = counts[7] = rows
    lengths[11], counts[11] = 2000, 1
    starts = [n - c for n, c in zip(lengths, counts)]
    pages = Pages(kc, 1, lengths, kv, page, hd, dtype)
    g = generator(4)
    pages.key.copy_(normal(g, *pages.key.shape))
    pages.value.copy_(normal(g, *pages.value.shape))
    q = normal(g, batch, rows, heads * hd)
    got = run_attention(kc, pages, q, starts, counts, heads, kv, hd)
    for b in range(batch):
        assert (got[b, counts[b]:] == -7).all()
    some = [7, 11] + [int(b) for b in rng.integers(0, batch, 60)]
    keep = [c if b in some else 0 for b, c in enumerate(counts)]
    want, top = attention_64(pages, q, starts, keep, heads, kv, hd, torch.full_like(q, -7.0))
    close(got[some], want[some], hd, top)


def test_attention_follows_the_contiguous_kernels(kc):
    """The same keys and values in a contiguous cache: k_attention_kv's result within both kernels' roundings."""
    heads, kv, hd, n = 32, 8, 128, 700
    pages = Pages(kc, 2, [n], kv, 64, hd, torch.float32)
    g = generator(12)
    fill_normal(pages, g, [n])
    keys, values = (x.float().contiguous() for x in pages.take(0, n))
    q = normal(g, 1, 1, heads * hd)
    got = run_attention(kc, pages, q, [n - 1], [1], heads, kv, hd)
    want = torch.empty(heads * hd, device="cuda")
    work = kc.attention_work(heads, kv, hd, n)
    kc.k_attention_kv(want, q, keys, values, work, heads, kv, hd, n, n - 1)
    kc.status()
    kc.k_attention_free(work)
    _, top = attention_64(pages, q, [n - 1], [1], heads, kv, hd, q)
    close(got.view(-1), want.double(), hd, 2 * top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=name_of)
def test_attention_offsets_past_32_bits(kc, dtype):
    """One request over a whole pool of more than 2^31 elements, its first and last pages the ones that count."""
    kv, hd, page, heads, n_pages = 8, 128, 64, 32, 33000
    key, value = (torch.zeros(n_pages, kv, page, hd, dtype=dtype, device="cuda") for _ in range(2))
    n = n_pages * page - 5
    table = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    g = generator(3)
    q = normal(g, 1, 1, heads * hd)
    big = normal(g, kv, hd).to(dtype)
    for p, scale in ((0, 1.0), (n - 1, 2.0), (n // 2, 3.0)):
        at = n_pages - 1 - p // page, slice(None), p % page
        key[at] = (40 * q.view(kv, heads // kv, hd)[:, 0] / hd ** 0.5).to(dtype)
        value[at] = (scale * big.float()).to(dtype)
    cache = kc.paged_cache(key, value, table)
    out = torch.empty_like(q)
    work = kc.paged_attention_work(heads, kv, hd, 1)
    kc.k_attention_paged_rows(out, None, None, q, cache, dev([n - 1]), None, work, heads, kv, hd, 1, 1, 0)
    assert kc.status() == 0
    want = torch.zeros(kv, heads // kv, hd, dtype=torch.float64, device="cuda")
    top = 1.0
    for h in range(kv):
        s = (q.view(kv, -1, hd)[h].double() @ key[:, h].flatten(0, 1).double().T) / hd ** 0.5
        order = (torch.arange(n_pages * page, device="cuda") // page * -page + (n_pages - 1) * page +
                 torch.arange(n_pages * page, device="cuda") % page)  # the position of each row of the pool
        s = torch.where(order < n, s, -float("inf"))
        top = max(top, float(s[s > -float("inf")].abs().max()))
        want[h] = s.softmax(-1) @ value[:, h].flatten(0, 1).double()
    close(out.view(kv, -1, hd), want, hd, top)


# ---- log probabilities -------------------------------------------------------------------------------------------------

def check_logprobs(x, tokens, top, got, skip=()):
    lp, ent, ids, best = got
    for r in range(x.shape[0]):
        if r in skip:
            continue
        row = x[r].double()
        p = torch.log_softmax(row, -1)
        w = p.exp()
        d = torch.where(w > 0, row.max() - row, 0.0)
        mean, square = float((w * d).sum()), float((w * d * d).sum())
        tol = lambda v: U * (v.abs() + mean + 12)  # noqa: E731
        order = torch.argsort(row, descending=True, stable=True)[:top]
        if top:
            assert torch.equal(ids[r].long(), order)
            finite = p[order] > -float("inf")
            assert torch.equal(best[r] > -float("inf"), finite)
            assert ((best[r].double() - p[order]).abs() <= tol(p[order]))[finite].all()
        if tokens is not None:
            want = p[tokens[r]]
            assert (lp[r] == want) if want == -float("inf") else (lp[r].double() - want).abs() <= tol(want)
        if ent is not None:
            want = float(torch.special.entr(w).sum())
            assert abs(float(ent[r]) - want) <= U * (want + square + 5 * mean + 12 * (1 + mean))


def run_logprobs(kc, x, tokens, top, vocab=None, entropy=True):
    rows = x.shape[0]
    lp = torch.full((rows,), -7.0, device="cuda") if tokens is not None else None
    ent = torch.full((rows,), -7.0, device="cuda") if entropy else None
    ids = torch.full((rows, top), -7, dtype=torch.int32, device="cuda") if top else None
    best = torch.full((rows, top), -7.0, device="cuda") if top else None
    kc.k_token_logprobs(lp, ent, ids, best, x, x.stride(0), dev(tokens), vocab or x.shape[1], rows, top)
    return lp, ent, ids, best


LOGPROBS = [(1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 33, 32), (1, 1000, 5), (70, 4099, 20), (3, 16384, 32),
            (2, 16385, 1), (9, 32000, 20), (300, 777, 5), (5, 50001, 0), (4, 128256, 20), (2, 262145, 32), (1, 700001, 20),
            (200, 128256, 8), (1, 128256, 0)]


@pytest.mark.parametrize("case", LOGPROBS, ids=lambda c: "-".join(map(str, c)))
def test_logprobs(kc, case):
    rows, vocab, top = case
    g = generator(vocab)
    x = 3 * normal(g, rows, vocab)
    tokens = [int(t) for t in np.random.default_rng(vocab).integers(0, vocab, rows)]
    got = run_logprobs(kc, x, tokens, top)
    assert kc.status() == 0
    check_logprobs(x, tokens, top, got)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("vocab", [130, 5001, 40003])
def test_logprobs_strides_and_alignment(kc, vocab, offset):
    """Rows that begin at any element; what lies between them is NaN."""
    rows, ld = 6, vocab + 5
    room = torch.full((rows * ld + offset + 8,), float("nan"), device="cuda")
    x = room[offset:offset + rows * ld].view(rows, ld)[:, :vocab]
    x.copy_(2 * normal(generator(vocab), rows, vocab))
    tokens = [0, vocab - 1, 5, 6, 7, 8]
    got = run_logprobs(kc, x, tokens, 7)
    assert kc.status() == 0
    check_logprobs(x, tokens, 7, got)


@pytest.mark.parametrize("vocab", [40, 3000, 60000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two", "zeros", "steps", "masked", "one", "block", "peaked",
                                  "large", "far"])
def test_logprobs_shapes_of_rows(kc, kind, vocab):
    """Ties of every number, orders that put the top ones together, masks, and rows near their ends of the range."""
    g = generator(vocab)
    at = torch.arange(vocab, device="cuda", dtype=torch.float32)
    inf = float("inf")
    row = {"equal": torch.full((vocab,), 1.25, device="cuda"), "rising": at / vocab * 9, "falling": -at / vocab * 9,
           "two": torch.where(at % 2 == 1, 3.0, 2.0), "zeros": torch.where(at % 3 == 1, -0.0, 0.0),
           "steps": torch.floor(at / 7) % 5, "masked": torch.where(at % 10 == 3, normal(g, vocab), -inf),
           "one": torch.where(at == vocab - 2, -5.0, -inf), "block": torch.where((at > 17) & (at < 36), 8.0 + at / 100, 0.0),
           "peaked": torch.where(at == 11, 30.0, 0.0) + normal(g, vocab), "large": 1e30 * normal(g, vocab),
           "far": torch.where(at == 3, 3e38, -3e38)}[kind]
    x = row[None].repeat(3, 1).contiguous()
    tokens, top = [int(row.argmax()), 0, vocab - 1], min(32, vocab)
    got = run_logprobs(kc, x, tokens, top)
    assert kc.status() == 0
    if kind in ("large", "far"):  # differences past fp32's range: the order, and the winner's certainty
        order = torch.argsort(row.double(), descending=True, stable=True)[:top]
        assert torch.equal(got[2], order.int().repeat(3, 1)) and float(got[0][0]) == 0.0 and float(got[1][0]) == 0.0
        assert (got[3][:, 0] == 0.0).all() and not torch.isnan(got[3]).any()
    else:
        check_logprobs(x, tokens, top, got)


@pytest.mark.parametrize("period", [2048, 4096])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_logprobs_many_candidates(kc, period, top):
    """The likeliest tokens all at a power of two from one another, more than any list of them has room for."""
    vocab = 128256
    at = torch.arange(vocab, device="cuda")
    x = torch.where(at % period < 80, 5.0 + torch.rand(vocab, device="cuda", generator=generator(1)), normal(generator(2), vocab))
    x = torch.stack([x, x.round(), torch.where(at % period < 80, 6.0, -1.0)]).contiguous()
    tokens = [0, 79, 128255]
    got = run_logprobs(kc, x, tokens, top)
    assert kc.status() == 0
    check_logprobs(x, tokens, top, got)


@pytest.mark.parametrize("rows,vocab,top", [(2048, 128256, 5), (1000, 60001, 20), (64, 128256, 20)])
def test_logprobs_many_rows_again_and_again(kc, rows, vocab, top):
    """Every row of many, with the memory busy: the stages of the ring are read before they are written again."""
    g = generator(vocab)
    inputs = [3 * normal(g, rows, vocab) for _ in range(2)]
    tokens = [int(t) for t in np.random.default_rng(rows).integers(0, vocab, rows)]
    at = dev(tokens).long()[:, None]
    want = []
    for x in inputs:
        p = torch.cat([torch.log_softmax(y.double(), -1).gather(1, t) for y, t in zip(x.split(256), at.split(256))])
        want.append((p[:, 0], torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top].int()))
    for i in range(12):
        lp, _, ids, _ = run_logprobs(kc, inputs[i % 2], tokens, top)
        p, order = want[i % 2]
        # three standard deviations of the logits cover the mean of d: E d <= 30
        assert ((lp.double() - p).abs() <= U * (p.abs() + 30 + 12)).all()
        assert torch.equal(ids, order)
    assert kc.status() == 0


def test_logprobs_small_differences_from_certainty(kc):
    """The likeliest token's log probability -e and the entropy of a row that is nearly certain keep their own digits."""
    vocab = 2000
    x = torch.zeros(5, vocab, device="cuda")
    for r, top in enumerate((12.0, 20.0, 30.0, 50.0, 80.0)):
        x[r, 77] = top
    lp, ent, _, best = run_logprobs(kc, x, [77] * 5, 3)
    # by the sum of the rest: 64-bit log_softmax rounds it against the 1 (-0 where -log(1 + 1999 e^-50) is -3.9e-19)
    d = torch.tensor([12.0, 20.0, 30.0, 50.0, 80.0], dtype=torch.float64, device="cuda")
    rest = (vocab - 1) * torch.exp(-d)
    p, h = -torch.log1p(rest), torch.log1p(rest) + rest * d / (1 + rest)
    # log(1 + s) = s - ..: no digit of s lost, s off by (d + 12) u of itself
    for got, want, extra in ((lp, p, 1), (best[:, 0], p, 1), (ent, h, 2)):
        assert ((got.double() - want).abs() <= extra * 100 * U * want.abs()).all()


def test_logprobs_rows_out_of_use(kc):
    x = normal(generator(1), 4, 5000)
    x[1], x[3] = float("nan"), float("nan")
    got = run_logprobs(kc, x, [5, -1, 4999, -1], 6)
    assert kc.status() == 0
    check_logprobs(x, [5, -1, 4999, -1], 6, got, skip=(1, 3))
    for y in got:
        assert (y[1] == -7).all() and (y[3] == -7).all()


@pytest.mark.parametrize("vocab", [50, 5000, 70000])
@pytest.mark.parametrize("wrong", ["nan", "inf", "empty", "token", "negative"])
def test_logprobs_reports(kc, wrong, vocab):
    for where in (0, vocab // 2, vocab - 1):
        x = normal(generator(2), 3, vocab)
        tokens = [1, 2, 3]
        if wrong == "nan":
            x[1, where] = float("nan")
        elif wrong == "inf":
            x[1, where] = float("inf")
        elif wrong == "empty":
            x[1] = -float("inf")
        else:
            tokens[1] = vocab + where if wrong == "token" else -2 - where
        got = run_logprobs(kc, x, tokens, 4)
        with pytest.raises(kc.KernelError):
            kc.status()
        check_logprobs(x, tokens, 4, got, skip=(1,))
        lp, ent, ids, best = got
        assert torch.isnan(lp[1]) and torch.isnan(ent[1]) and (ids[1] == -1).all() and torch.isnan(best[1]).all()


def test_logprobs_parts(kc):
    """Without tokens, without entropy, without top tokens."""
    x = normal(generator(3), 3, 9000)
    got = run_logprobs(kc, x, None, 5)
    assert kc.status() == 0
    check_logprobs(x, None, 5, got)
    got = run_logprobs(kc, x, [1, 2, 3], 0, entropy=False)
    assert kc.status() == 0
    check_logprobs(x, [1, 2, 3], 0, got)


def test_logprobs_offsets_past_32_bits(kc):
    rows, vocab = 17000, 128256
    x = torch.zeros(rows, vocab, device="cuda")
    assert x.numel() > 2 ** 31
    x[-1] = 3 * normal(generator(4), vocab)
    tokens = [-1] * (rows - 1) + [777]
    got = run_logprobs(kc, x, tokens, 20)
    assert kc.status() == 0
    check_logprobs(x[-1:], [777], 20, [y[-1:] for y in got])


# ---- together ----------------------------------------------------------------------------------------------------------

def serving(kc, dtype, seed=0):
    """Three requests of one layer's width over a paged cache: one decodes, one brings two drafts, one its prompt."""
    dim, heads, kv, hd, vocab, B, R, page, gs = 512, 8, 2, 64, 1000, 3, 6, 16, 64
    g = generator(seed)
    lengths = [100, 37, 0]
    pages = Pages(kc, seed, [n + R for n in lengths], kv, page, hd, dtype)
    fill_normal(pages, g, lengths)
    weight = lambda n, k: (torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8),  # noqa: E731
                           torch.rand(n, k // gs, device="cuda", generator=g) * 0.002)
    s = dict(pages=pages, x=normal(g, B * R, dim), norm=1 + 0.1 * normal(g, dim), wq=weight(heads * hd, dim),
             wk=weight(kv * hd, dim), wv=weight(kv * hd, dim), wo=weight(dim, heads * hd), cls=weight(vocab, dim),
             starts=dev(lengths), counts=dev([1, 3, 6]), rope=rope_table(256, hd),
             work=kc.paged_attention_work(heads, kv, hd, B, R), tokens=dev([int(t) for t in range(5, 5 + B * R)]))
    z = lambda *shape, t=torch.float32: torch.zeros(*shape, dtype=t, device="cuda")  # noqa: E731
    s.update(xq=z(B * R, dim, t=torch.int8), xs=z(B * R, dim // gs), qkv=z(B * R, (heads + 2 * kv) * hd),
             q=z(B, R, heads * hd), att=z(B, R, heads * hd), oq=z(B, R, heads * hd, t=torch.int8),
             os=z(B, R, heads * hd // gs), y=z(B * R, dim), yq=z(B * R, dim, t=torch.int8), ys=z(B * R, dim // gs),
             logits=z(B * R, vocab), lp=z(B * R), ent=z(B * R), ids=z(B * R, 5, t=torch.int32), best=z(B * R, 5))
    s.update(dim=dim, heads=heads, kv=kv, hd=hd, vocab=vocab, B=B, R=R, gs=gs)
    return s


def step(kc, s):
    """QKV, rotation and storing, attention with its output quantized, Wo, classifier, log probabilities."""
    heads, kv, hd, B, R, gs, dim = (s[n] for n in ("heads", "kv", "hd", "B", "R", "gs", "dim"))
    ld = (heads + 2 * kv) * hd
    q, k, v = s["qkv"][:, :heads * hd], s["qkv"][:, heads * hd:(heads + kv) * hd], s["qkv"][:, (heads + kv) * hd:]
    kc.k_rmsnorm_q8_rows(s["xq"], s["xs"], None, s["x"], dim, s["norm"], B * R, dim, 1e-5, gs)
    kc.k_gemm_q8(s["xq"], s["xs"], B * R, dim, gs, [kc.segment(c, w, ldc=ld) for c, w in
                                                   ((q, s["wq"]), (k, s["wk"]), (v, s["wv"]))])
    kc.k_rope_kv_store_paged(s["q"], heads * hd, q, ld, k, v, ld, s["pages"].cache, s["rope"], 256, s["starts"], s["counts"],
                             heads, kv, hd, B, R)
    kc.k_attention_paged_rows(s["att"], s["oq"], s["os"], s["q"], s["pages"].cache, s["starts"], s["counts"], s["work"], heads,
                              kv, hd, B, R, gs)
    kc.k_gemm_q8(s["oq"], s["os"], B * R, heads * hd, gs, [kc.segment(s["y"], s["wo"])])
    kc.k_rmsnorm_q8_rows(s["yq"], s["ys"], None, s["y"], dim, s["norm"], B * R, dim, 1e-5, gs)
    kc.k_gemm_q8(s["yq"], s["ys"], B * R, dim, gs, [kc.segment(s["logits"], s["cls"])])
    kc.k_token_logprobs(s["lp"], s["ent"], s["ids"], s["best"], s["logits"], s["vocab"], s["tokens"], s["vocab"], B * R, 5)


def check_step(kc, s, starts, counts):
    """Each operator's outputs from the inputs that the step gave it."""
    heads, kv, hd, B, R = (s[n] for n in ("heads", "kv", "hd", "B", "R"))
    pages = s["pages"]
    for b in range(B):
        for r in range(counts[b]):
            row, p = s["qkv"][b * R + r], starts[b] + r
            at, slot = int(pages.table[b, p // pages.page]), p % pages.page
            assert same(s["q"][b, r], rotate(row[:heads * hd], s["rope"][p], hd).flatten())
            assert same(pages.key[at, :, slot], rotate(row[heads * hd:(heads + kv) * hd], s["rope"][p], hd).to(pages.key.dtype))
            assert same(pages.value[at, :, slot], row[(heads + kv) * hd:].view(kv, hd).to(pages.key.dtype))
    want, top = attention_64(pages, s["q"], starts, counts, heads, kv, hd, s["att"])
    close(s["att"], want, hd, top)
    check_logprobs(s["logits"], s["tokens"].tolist(), 5, (s["lp"], s["ent"], s["ids"], s["best"]))


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_a_step_over_a_paged_cache(kc, dtype):
    s = serving(kc, dtype)
    step(kc, s)
    assert kc.status() == 0
    check_step(kc, s, [100, 37, 0], [1, 3, 6])


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_captured_steps(kc, dtype):
    """A captured step replays as requests grow and get pages, on a stream of its own, between eager calls."""
    s = serving(kc, dtype, 1)
    step(kc, s)  # sizes every buffer that a first call makes
    assert kc.status() == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(kc, s)
        starts, counts = [101, 40, 6], [1, 2, 0]
        for i in range(4):
            s["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
            s["counts"].copy_(torch.tensor(counts, dtype=torch.int32))
            s["x"].copy_(normal(generator(i), *s["x"].shape))
            graph.replay()
            side.synchronize()
            check_step(kc, s, starts, counts)
            starts = [n + c for n, c in zip(starts, counts)]
            counts = [1, 1, 1]
            if i == 1:  # an eager call of other sizes on the same work
                step(kc, s)
        assert kc.status() == 0


def test_two_works_on_two_streams(kc):
    """Two batches at once, a work each."""
    heads, kv, hd, n = 32, 8, 128, 900
    streams, states = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        pages = Pages(kc, i, [n] * 4, kv, 16, hd, torch.bfloat16)
        fill_normal(pages, generator(i), [n] * 4)
        q = normal(generator(10 + i), 4, 1, heads * hd)
        states.append((pages, q, torch.zeros_like(q), kc.paged_attention_work(heads, kv, hd, 4), dev([n - 1] * 4)))
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (pages, q, out, work, starts) in zip(streams, states):
            with torch.cuda.stream(stream):
                kc.k_attention_paged_rows(out, None, None, q, pages.cache, starts, None, work, heads, kv, hd, 4, 1, 0)
    torch.cuda.synchronize()
    assert kc.status() == 0
    for pages, q, out, _, _ in states:
        want, top = attention_64(pages, q, [n - 1] * 4, [1] * 4, heads, kv, hd, q)
        close(out, want, hd, top)


def test_one_work_for_batches_of_many_shapes(kc):
    """A work made for 12 rows of 32 heads serves every split of fewer rows, one after another, in any order of types."""
    work = kc.paged_attention_work(32, 8, 128, 4, 3)
    for i, (B, R, kv, dtype) in enumerate([(12, 1, 8, torch.bfloat16), (1, 12, 8, torch.float32), (4, 3, 4, torch.float16),
                                           (2, 5, 32, torch.bfloat16), (3, 4, 1, torch.float16), (12, 1, 8, torch.float32)]):
        lengths = [30 + 200 * ((i + b) % 4) for b in range(B)]
        pages = Pages(kc, i, lengths, kv, 16, 128, dtype)
        g = generator(i)
        fill_normal(pages, g, lengths)
        q = normal(g, B, R, 32 * 128)
        starts = [n - R for n in lengths]
        got = run_attention(kc, pages, q, starts, [R] * B, 32, kv, 128, work=work)
        want, top = attention_64(pages, q, starts, [R] * B, 32, kv, 128, q)
        close(got, want, 128, top)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_results_repeat(kc, dtype):
    """The same call gives the same bits, whichever share of a segment is done last."""
    heads, kv, hd, lengths = 32, 8, 128, [3000, 17, 640]
    pages = Pages(kc, 1, lengths, kv, 24, hd, dtype)
    g = generator(1)
    fill_normal(pages, g, lengths)
    q = normal(g, 3, 1, heads * hd)
    work = kc.paged_attention_work(heads, kv, hd, 3)
    first = run_attention(kc, pages, q, [n - 1 for n in lengths], None, heads, kv, hd, work=work)
    for _ in range(20):
        assert same(run_attention(kc, pages, q, [n - 1 for n in lengths], None, heads, kv, hd, work=work), first)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_nothing_in_use(kc, dtype):
    """No request uses a row: nothing is written, whatever the tables, starts and inputs hold."""
    heads, kv, hd, B, R = 8, 2, 64, 5, 3
    pages = Pages(kc, 1, [0] * B, kv, 16, hd, dtype, width=4)
    nan = torch.full((B, R, heads * hd), float("nan"), device="cuda")
    out, rope = torch.full_like(nan, -7.0), rope_table(64, hd)
    starts, counts = [-5, 1 << 30, 0, 7, -(1 << 31)], [0] * B
    assert run_store(kc, pages, nan, nan[..., :kv * hd], nan[..., :kv * hd], rope, starts, counts, heads, kv, hd, out) == 0
    run_attention(kc, pages, nan, starts, counts, heads, kv, hd, out=out)
    assert (out == -7).all() and torch.isnan(pages.key.float()).all() and torch.isnan(pages.value.float()).all()
    got = run_logprobs(kc, nan[0], [-1] * R, 4)
    assert kc.status() == 0 and all((x == -7).all() for x in got)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_the_librarys_own_memory_and_plain_launches(kc, dtype):
    """A work on memory that the library allocates; launches without programmatic dependence."""
    import ctypes
    heads, kv, hd, lengths = 8, 2, 128, [300, 5]
    pages = Pages(kc, 1, lengths, kv, 16, hd, dtype)
    g = generator(1)
    fill_normal(pages, g, lengths)
    q = normal(g, 2, 1, heads * hd)
    work = kc.AttentionWork()
    kc._call("k_attention_paged_init", ctypes.byref(work), heads, kv, hd, 2, 1, None)
    assert work.external == 0
    starts = [n - 1 for n in lengths]
    want, top = attention_64(pages, q, starts, [1, 1], heads, kv, hd, q)
    kc.load().kernels_set_pdl(0)
    try:
        for _ in range(3):
            close(run_attention(kc, pages, q, starts, None, heads, kv, hd, work=work), want, hd, top)
        x = 3 * normal(g, 5, 40000)
        got = run_logprobs(kc, x, [1, 2, 3, 4, 5], 7)
        assert kc.status() == 0
        check_logprobs(x, [1, 2, 3, 4, 5], 7, got)
    finally:
        kc.load().kernels_set_pdl(1)
        kc.k_attention_free(work)


def test_a_product_before_and_behind(kc):
    """Attention between tensor-core products that start while it runs: back to back, many times, the same bits."""
    s = serving(kc, torch.bfloat16, 5)
    step(kc, s)
    assert kc.status() == 0
    first = [s[n].clone() for n in ("att", "logits", "lp", "ids")]
    for _ in range(50):
        step(kc, s)
    assert kc.status() == 0
    for x, n in zip(first, ("att", "logits", "lp", "ids")):
        assert torch.equal(x, s[n])


def test_mirror_refuses_what_does_not_fit(kc):
    z = lambda *shape, t=torch.float32: torch.zeros(*shape, dtype=t, device="cuda")  # noqa: E731
    key, table = z(4, 2, 16, 64, t=torch.bfloat16), z(3, 4, t=torch.int32)
    for k, v, t in ((key, key.half(), table), (key.double(), key.double(), table), (key.transpose(2, 3), key.transpose(2, 3), table),
                    (key, key[:3], table), (key, key, table.long()), (key, key, table.cpu()), (key.cpu(), key, table),
                    (key[0], key[0], table), (key, key, table[0]), (key, z(8, 2, 16, 64, t=torch.bfloat16)[::2], table)):
        with pytest.raises(kc.KernelError):
            kc.paged_cache(k, v, t)
    cache = kc.paged_cache(key, key.clone(), table)
    q, out, starts = z(3, 1, 512), z(3, 1, 512), z(3, t=torch.int32)
    work = kc.paged_attention_work(8, 2, 64, 3)
    call = lambda out=out, q=q, cache=cache, starts=starts, heads=8, kv=2, hd=64, batch=3: kc.k_attention_paged_rows(  # noqa: E731
        out, None, None, q, cache, starts, None, work, heads, kv, hd, batch, 1, 0)
    for bad in (dict(out=out.half()), dict(q=q.cpu()), dict(starts=starts.long()), dict(kv=4), dict(hd=32), dict(batch=4),
                dict(q=z(512, 3, 1).transpose(0, 1))):
        with pytest.raises(kc.KernelError):
            call(**bad)
    store = lambda q=q, kv=z(3, 1, 128), rope=z(8, 128), counts=None: kc.k_rope_kv_store_paged(  # noqa: E731
        out, 512, q, 512, kv, kv, 128, cache, rope, 8, starts, counts, 8, 2, 64, 3, 1)
    for bad in (dict(q=q.bfloat16()), dict(kv=z(3, 1, 128).cpu()), dict(rope=z(128, 8).T), dict(counts=starts.long())):
        with pytest.raises(kc.KernelError):
            store(**bad)
    x, tokens = z(3, 100), z(3, t=torch.int32)
    for bad in (dict(x=x.half()), dict(x=x.T.contiguous().T), dict(tokens=tokens.long()), dict(lp=z(3).double())):
        args = dict(dict(x=x, tokens=tokens, lp=z(3)), **bad)
        with pytest.raises(kc.KernelError):
            kc.k_token_logprobs(args["lp"], None, None, None, args["x"], 100, args["tokens"], 100, 3, 0)
    assert kc.status() == 0


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 256), (torch.bfloat16, 96), (torch.float16, 33), (torch.float32, 64),
                                      (torch.bfloat16, 128)], ids=str)
@pytest.mark.parametrize("page", [-2, -3, -128, 67])
def test_attention_reports_every_number_that_is_no_page(kc, page, dtype, hd):
    """Small negative numbers, and the first one past the pool, are pages as little as any other."""
    heads, kv, n = 8, 2, 60
    pages = Pages(kc, 3, [n, n], kv, 2, hd, dtype, spare=7)
    assert pages.key.shape[0] == 67
    g = generator(3)
    fill_normal(pages, g, [n, n])
    q = normal(g, 2, 1, heads * hd)
    want, top = attention_64(pages, q, [n - 1] * 2, [1, 1], heads, kv, hd, q)
    for index in (0, 11, 29):
        pages.device_table[1, index] = page
        out = torch.full_like(q, -7.0)
        with pytest.raises(kc.KernelError):
            run_attention(kc, pages, q, [n - 1] * 2, [1, 1], heads, kv, hd, out=out)
        assert (out[1] == -7).all()
        close(out[:1], want[:1], hd, top)
        pages.device_table[1, index] = int(pages.table[1, index])


@pytest.mark.parametrize("batch", [1, 5, 128])
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 256), (torch.bfloat16, 96), (torch.float16, 33), (torch.float32, 64),
                                      (torch.bfloat16, 128)], ids=str)
def test_attention_bad_first_pages_every_time(kc, dtype, hd, batch):
    """A share whose first page is none: what the first fetch of any warp finds is reported, call after call."""
    heads, kv, n, times = 8, 2, 3, 50
    pages = Pages(kc, 3, [n] * batch, kv, 1, hd, dtype)
    g = generator(3)
    fill_normal(pages, g, [n] * batch)
    q = normal(g, batch, 1, heads * hd)
    work, starts = kc.paged_attention_work(heads, kv, hd, batch), dev([n - 1] * batch)
    good = pages.device_table.clone()
    outs = torch.full((times, batch, 1, heads * hd), -7.0, device="cuda")
    want, top = attention_64(pages, q, [n - 1] * batch, [1] * batch, heads, kv, hd, q)
    bad = [i % batch for i in range(times)]
    for i in range(times):
        pages.device_table.copy_(good)
        pages.device_table[bad[i], i % n] = -1 - i
        kc.k_attention_paged_rows(outs[i], None, None, q, pages.cache, starts, None, work, heads, kv, hd, batch, 1, 0)
        with pytest.raises(kc.KernelError):
            kc.status()
    for i in range(times):
        others = [b for b in range(batch) if b != bad[i]]
        assert (outs[i, bad[i]] == -7).all()
        if others:
            close(outs[i, others], want[others], hd, top)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("vocab", list(range(1, 13)) + [4096, 4097, 4098, 4099, 8191, 262143, 262145])
def test_logprobs_at_the_ends_of_rows(kc, vocab, offset):
    """The likeliest tokens, the largest of them among equals, and the tokens asked for are a row's first and last ones, whose
    16 bytes are not all the row's; what lies there beside them is NaN or larger than any."""
    rows = 4
    ld = vocab + 7
    room = torch.full((rows * ld + offset,), float("nan"), device="cuda")
    room[::2] = float("inf")
    x = room[offset:].as_strided((rows, vocab), (ld, 1))
    g = generator(vocab + offset)
    base = normal(g, rows, vocab)
    ends = [i for i in range(vocab) if i < 4 or i >= vocab - 4]
    base[0, ends] = 6.0 + 0.1 * torch.rand(len(ends), device="cuda", generator=g)
    base[1, ends] = 7.0
    base[2, ends[-1]] = 30.0
    base[3, ends[0]] = 30.0
    x.copy_(base)
    top = min(vocab, 8)
    for tokens in ([0, vocab - 1, vocab - 1, 0], [vocab // 2] * 4):
        got = run_logprobs(kc, x, tokens, top)
        assert kc.status() == 0
        check_logprobs(base, tokens, top, got)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_captured_steps_with_new_and_moved_pages(kc, dtype):
    """A captured step replays while a request reaches a page that was none at capture and gets it only then, and while pages
    that are in use move elsewhere in the pool."""
    s = serving(kc, dtype, 2)
    page = 16
    pages = s["pages"] = Pages(kc, 2, [106, 43, 6], s["kv"], page, s["hd"], dtype, width=9, spare=8)  # the rest: no page
    fill_normal(pages, generator(2), [100, 37, 0])
    step(kc, s)  # sizes every buffer that a first call makes
    assert kc.status() == 0
    used = set(pages.table[0, :7]) | set(pages.table[1, :3]) | {pages.table[2, 0]}
    spare = [p for p in range(pages.key.shape[0]) if p not in used]
    none = lambda b, index: not 0 <= pages.table[b, index] < pages.key.shape[0]  # noqa: E731
    assert none(0, 7) and none(2, 1)

    def point(b, index, to):  # the table's entry, here and on the device
        pages.table[b, index] = to
        pages.device_table[b, index] = to

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    starts, counts = [101, 40, 6], [6, 1, 6]
    with torch.cuda.stream(side):
        s["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
        s["counts"].copy_(torch.tensor(counts, dtype=torch.int32))
        with torch.cuda.graph(graph, stream=side):
            step(kc, s)
        for i in range(4):
            if starts[0] + counts[0] > 7 * page and none(0, 7):
                point(0, 7, spare.pop())
            if starts[2] + counts[2] > page and none(2, 1):
                point(2, 1, spare.pop())
            if i >= 2:  # the first page of request 1 moves, and what it held is overwritten
                old, new = int(pages.table[1, 0]), spare.pop()
                for cache in (pages.key, pages.value):
                    cache[new] = cache[old]
                    cache[old] = float("nan")
                point(1, 0, new)
            s["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
            s["counts"].copy_(torch.tensor(counts, dtype=torch.int32))
            s["x"].copy_(normal(generator(i), *s["x"].shape))
            graph.replay()
            side.synchronize()
            assert kc.status() == 0
            check_step(kc, s, starts, counts)
            starts = [n + c for n, c in zip(starts, counts)]
            counts = [5, 1, 5] if i == 0 else [1, 2, 3]
        assert starts[0] > 7 * page and starts[2] > page


def unsound_batch(kc, seed, batch, rows, kv, page, hd, dtype):
    """A batch of short requests, some without rows, and of those with rows some with an unsound start or count or a page
    that is none: (pages, starts, counts, counts of the sound ones)."""
    rng = np.random.default_rng(seed)
    counts = [int(c) for c in rng.integers(0, rows + 1, batch)]
    lengths = [c + int(rng.integers(0, 70)) if c else 0 for c in counts]
    starts = [n - c for n, c in zip(lengths, counts)]
    pages = Pages(kc, seed, lengths, kv, page, hd, dtype)
    g = generator(seed)
    fill_normal(pages, g, lengths)
    live = [b for b in range(batch) if counts[b]]
    wrong = sorted(rng.choice(live, 24, replace=False).tolist()) + [live[0], live[-1]]
    sound = [0 if b in wrong else c for b, c in enumerate(counts)]
    most = pages.width * page
    for i, b in enumerate(wrong):
        if i % 6 == 0:
            starts[b] = -1 - i
        elif i % 6 == 1:
            starts[b] = most - counts[b] + 1
        elif i % 6 == 2:
            counts[b] = rows + 1 + i
        elif i % 6 == 3:
            counts[b] = -1 - i
        elif i % 6 == 4:
            starts[b] = 2 ** 31 - 1
        else:
            pages.device_table[b, int(rng.integers(0, -(-lengths[b] // page)))] = -1 - i
    return pages, starts, counts, sound


@pytest.mark.parametrize("batch,rows", [(129, 3), (400, 1), (1000, 2)])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.float32, 128),
                                      (torch.bfloat16, 96), (torch.float32, 256)], ids=str)
def test_attention_many_requests_some_unsound(kc, dtype, hd, batch, rows):
    """More requests than a warp looks at alone, unsound ones among them: an error, their rows as they were, the others'
    right, and the work as good as new."""
    heads, kv, page = 8, 2, 16
    pages, starts, counts, sound = unsound_batch(kc, batch + hd, batch, rows, kv, page, hd, dtype)
    q = normal(generator(1), batch, rows, heads * hd)
    work = kc.paged_attention_work(heads, kv, hd, batch, rows)
    out = torch.full_like(q, -7.0)
    want, top = attention_64(pages, q, starts, sound, heads, kv, hd, torch.full_like(q, -7.0))
    with pytest.raises(kc.KernelError):
        run_attention(kc, pages, q, starts, counts, heads, kv, hd, work=work, out=out)
    for b in range(batch):
        assert (out[b, sound[b]:] == -7).all()
    close(out, want, hd, top)
    # Another batch to the kernel, whose work is shared out without them: equal results, not equal bits.
    close(run_attention(kc, pages, q, starts, sound, heads, kv, hd, work=work), want, hd, top)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
def test_store_many_requests_some_unsound(kc, dtype):
    heads, kv, hd, batch, rows, page = 4, 2, 64, 300, 3, 16
    pages, starts, counts, sound = unsound_batch(kc, 5, batch, rows, kv, page, hd, dtype)
    g = generator(2)
    q, k, v = (normal(g, batch, rows, n * hd) for n in (heads, kv, kv))
    rope, q_out = rope_table(pages.width * page, hd), torch.full((batch, rows, heads * hd), -7.0, device="cuda")
    # A row whose page is none is left out, and only that row; a request that is unsound whole.
    table, most = pages.device_table.tolist(), pages.width * page
    tried = [c if 0 <= c <= rows and 0 <= s <= most - c else 0 for s, c in zip(starts, counts)]
    left = {(b, r) for b in range(batch) for r in range(tried[b])
            if not 0 <= table[b][(starts[b] + r) // page] < pages.key.shape[0]}
    want = stored(pages, q, k, v, rope, starts, tried, heads, kv, hd, q_out, skip=left)
    with pytest.raises(kc.KernelError):
        run_store(kc, pages, q, k, v, rope, starts, counts, heads, kv, hd, q_out)
    check_store((q_out, pages.key, pages.value), want)


@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (32, 8, 64), (28, 4, 128), (8, 2, 96)])
@pytest.mark.parametrize("rows", [5, 8, 150])
def test_attention_prompts_drafts_and_single_tokens_together(kc, heads, kv, hd, rows, dtype):
    """One call of a serving batch: a prompt or drafts of the longest number of rows, drafts, single tokens, and a slot out of
    use; each request as in a call of its own."""
    counts = [1, rows, 1, 0, 3, 1, 1, 2, 1]
    starts = [500, 0, 1, 0, 130, 77, 1023, 64, 0]
    lengths = [s + c if c else 0 for s, c in zip(starts, counts)]
    pages = Pages(kc, rows, lengths, kv, 16, hd, dtype)
    g = generator(hd + rows)
    fill_normal(pages, g, lengths)
    q = 1.5 * normal(g, len(counts), rows, heads * hd)
    got = run_attention(kc, pages, q, starts, counts, heads, kv, hd)
    want, top = attention_64(pages, q, starts, counts, heads, kv, hd, torch.full_like(q, -7.0))
    for b, c in enumerate(counts):
        assert (got[b, c:] == -7).all()
    close(got, want, hd, top)
    for b, c in enumerate(counts):
        if c:
            alone = Pages.__new__(Pages)
            alone.__dict__.update(pages.__dict__)
            alone.table, alone.device_table = pages.table[b:b + 1], pages.device_table[b:b + 1].contiguous()
            alone.cache = kc.paged_cache(pages.key, pages.value, alone.device_table)
            own = run_attention(kc, alone, q[b:b + 1, :c].contiguous(), [starts[b]], [c], heads, kv, hd)
            close(own, want[b:b + 1, :c], hd, top)


@pytest.mark.parametrize("hd", [128, 64, 96])
@pytest.mark.parametrize("dtype", TYPES, ids=name_of)
@pytest.mark.parametrize("bits", [20, 28, 31])
def test_attention_small_weights_keep_their_digits(kc, dtype, hd, bits):
    """A weight of 2^-bits of the row's largest, the only one with a value: the result is its product, to fp32's roundings."""
    heads, kv, n = 4, 1, 300
    pages = Pages(kc, 5, [n], kv, 16, hd, dtype)
    keys, values = torch.zeros(kv, n, hd, device="cuda"), torch.zeros(kv, n, hd, device="cuda")
    keys[:, :, 0] = 8.0
    keys[:, 130, 0] = 0.0
    values[:, 130] = 1.0 + torch.rand(hd, device="cuda", generator=generator(bits))
    pages.fill(0, keys, values)
    q = torch.zeros(1, 1, heads, hd, device="cuda")
    q[..., 0] = bits * float(np.log(2.0)) / 8.0 * hd ** 0.5
    q = q.view(1, 1, heads * hd)
    got = run_attention(kc, pages, q, [n - 1], [1], heads, kv, hd)
    want, top = attention_64(pages, q, [n - 1], [1], heads, kv, hd, q)
    assert 2.0 ** -(bits + 10) < float(want.abs().min()) and float(want.abs().max()) < 2.0 ** -(bits + 6)
    close(got, want, hd, top)
