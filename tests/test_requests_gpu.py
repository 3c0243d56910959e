"""GPU tests of the operators that serve a batch of requests over one prompt, against plain 64-bit forms of their
definitions.

Tolerances, from the number of roundings (fp32: half a step is u = 2^-24 of the value), each taken as random:
  - attention: a score is a chain of head_dim roundings of values up to the largest score S, about sqrt(head_dim) u S off;
    a score off by e moves a weight by e of itself, and weights, sums and joins add a few u. Four standard deviations:
    4 u (sqrt(head_dim) S + 8) of the largest output, per element.
  - adapters: with |B| |A| |x| the products' sum of magnitudes, 4 u (sqrt(n) + sqrt(rank) + 4) of it, per element, and
    2 u of base and result.
  - verification: whole numbers, equal.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CUDA = dict(device="cuda")


def normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ---- attention over a shared prefix ------------------------------------------------------------------------------------

def attention_64(q, pk, pv, prefix, k, v, starts, counts, heads, kv, hd, before):
    """Per request and row, in 64 bits; `before` where nothing is written. Also the largest score."""
    out, top = before.double().clone(), 1.0
    B, R = q.shape[:2]
    for b in range(B):
        for r in range(counts[b]):
            n = starts[b] + r + 1
            keys = torch.cat([pk[:, :prefix], k[b, :, :n]], 1).double()
            values = torch.cat([pv[:, :prefix], v[b, :, :n]], 1).double()
            s = torch.einsum("kgd,kpd->kgp", q[b, r].double().view(kv, heads // kv, hd), keys) / hd ** 0.5
            top = max(top, float(s.abs().max()))
            out[b, r] = torch.einsum("kgp,kpd->kgd", s.softmax(-1), values).reshape(-1)
    return out, top


def run_attention(kc, q, pk, pv, prefix, k, v, starts, counts, heads, kv, hd, out=None, gs=0, work=None):
    B, R = q.shape[:2]
    out = torch.full_like(q, -7.0) if out is None else out
    oq = torch.full(q.shape, 99, dtype=torch.int8, device="cuda") if gs else None
    os_ = torch.full((B, R, heads * hd // gs), -1.0, device="cuda") if gs else None
    mine = work or kc.shared_attention_work(heads, kv, hd, B, R)
    dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    try:
        kc.k_attention_shared_rows(out, oq, os_, q, pk, pv, pk.shape[1] if pk is not None else 0, prefix, k, v, dev(starts),
                                   dev(counts), mine, heads, kv, hd, k.shape[2], B, R, gs)
        kc.status()
    finally:
        if work is None:
            kc.k_attention_free(mine)
    return (out, oq, os_) if gs else out


def close(got, want, hd, top):
    tol = 4 * U * (hd ** 0.5 * top + 8) * max(float(want.abs().max()), 1e-30)
    assert float((got.double() - want).abs().max()) <= tol


ATTENTION = [  # heads, kv, hd, batch, rows, prefix, prefix room, own cache
    (1, 1, 64, 1, 1, 0, 0, 1),
    (1, 1, 64, 1, 1, 1, 1, 1),
    (8, 2, 128, 1, 1, 63, 64, 5),
    (8, 2, 128, 2, 3, 65, 80, 70),
    (32, 8, 128, 5, 4, 129, 130, 33),
    (32, 8, 64, 3, 2, 1000, 1000, 17),
    (32, 8, 64, 40, 5, 257, 300, 9),
    (16, 16, 64, 9, 1, 130, 131, 200),
    (14, 2, 64, 7, 8, 321, 321, 129),
    (28, 4, 128, 6, 7, 515, 520, 260),
    (8, 2, 32, 11, 3, 200, 203, 66),
    (6, 2, 48, 3, 2, 77, 78, 20),
    (12, 3, 96, 4, 3, 140, 150, 31),
    (4, 1, 256, 2, 2, 70, 71, 40),
    (6, 3, 10, 3, 4, 45, 46, 12),
    (2, 1, 33, 2, 2, 37, 40, 9),
    (48, 1, 128, 2, 3, 200, 200, 10),
]


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(map(str, c)))
def test_shared_attention(kc, case):
    heads, kv, hd, B, R, prefix, room, S = case
    g = generator(heads * 1000 + prefix)
    rng = np.random.default_rng(prefix + B)
    q, k, v = 1.5 * normal(g, B, R, heads * hd), normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    pk, pv = (normal(g, kv, room, hd), normal(g, kv, room, hd)) if room else (None, None)
    counts = [int(c) for c in rng.integers(0, min(R, S) + 1, B)]
    counts[-1] = min(R, S)
    starts = [int(rng.integers(0, S - c + 1)) for c in counts]
    starts[-1] = S - counts[-1]
    # What no row sees is NaN: behind the prefix and behind each request's last position, and the unused requests whole.
    if room:
        pk[:, prefix:], pv[:, prefix:] = float("nan"), float("nan")
    for b in range(B):
        seen = starts[b] + counts[b] if counts[b] else 0
        k[b, :, seen:], v[b, :, seen:] = float("nan"), float("nan")
        q[b, counts[b]:] = float("nan")
    got = run_attention(kc, q, pk, pv, prefix, k, v, starts, counts, heads, kv, hd)
    empty = torch.zeros(kv, 0, hd, device="cuda")
    want, top = attention_64(q, empty if pk is None else pk, empty if pv is None else pv, prefix, k, v, starts, counts,
                             heads, kv, hd, torch.full_like(q, -7.0))
    close(got, want, hd, top)
    for b in range(B):
        assert (got[b, counts[b]:] == -7.0).all()


@pytest.mark.parametrize("scale_k,scale_v", [(1e4, 1.0), (1.0, 1e6), (1e-6, 1e-20), (1e10, 1e20)])
def test_shared_attention_ranges(kc, scale_k, scale_v):
    """Keys and values far outside a half-precision number's range, and of mixed sizes within a cache; the queries are
    scaled the other way, so that the scores stay ordinary."""
    heads, kv, hd, B, R, prefix, S = 8, 2, 64, 2, 2, 200, 70
    g = generator(5)
    q = normal(g, B, R, heads * hd) / scale_k
    pk, k = normal(g, kv, prefix, hd) * scale_k, normal(g, B, kv, S, hd) * scale_k
    pv, v = normal(g, kv, prefix, hd) * scale_v, normal(g, B, kv, S, hd) * scale_v
    pk[:, :64] *= 1e-3  # a stretch of small keys, one of small values, one of large values far in
    pv[:, 64:128] *= 1e-4
    v[:, :, 64:] *= 1e3
    got = run_attention(kc, q, pk, pv, prefix, k, v, [S - R] * B, [R] * B, heads, kv, hd)
    want, top = attention_64(q, pk, pv, prefix, k, v, [S - R] * B, [R] * B, heads, kv, hd, got)
    close(got, want, hd, top)


def test_shared_attention_peaked_and_rising_scores(kc):
    """Scores that rise along the prefix (the running maximum moves in every tile) and ones with a single winner."""
    heads, kv, hd, B, R, prefix, S = 4, 1, 128, 3, 1, 700, 16
    g = generator(6)
    q = torch.ones(B, R, heads * hd, device="cuda")
    rise = torch.linspace(-40, 40, prefix, device="cuda")[None, :, None] / hd ** 0.5
    pk = rise.expand(kv, prefix, hd).contiguous()
    pv, k, v = normal(g, kv, prefix, hd), normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    for keys in (pk, pk.flip(1).contiguous(), torch.where(torch.arange(prefix, device="cuda")[:, None] == 333, 8.0, -8.0)
                 .expand(kv, prefix, hd).contiguous()):
        got = run_attention(kc, q, keys, pv, prefix, k, v, [S - 1] * B, [1] * B, heads, kv, hd)
        want, top = attention_64(q, keys, pv, prefix, k, v, [S - 1] * B, [1] * B, heads, kv, hd, got)
        close(got, want, hd, top)


@pytest.mark.parametrize("hd", [128, 64, 96, 256, 33])
@pytest.mark.parametrize("wrong", [float("nan"), float("inf"), float("-inf")])
def test_shared_attention_keeps_to_what_a_row_sees(kc, hd, wrong):
    """Positions that are not finite, in the keys or in the values: behind the prefix and the last row, where nobody sees
    them, and at the place of a later row of the same request, which alone has no result then; queries that are not
    finite spoil their own row only."""
    heads, kv, B, R, prefix, S = 8, 2, 5, 3, 130, 90
    starts, counts = [0, 61, 66, 10, 40], [3, 3, 3, 2, 1]
    g = generator(12)
    q, pk, pv = normal(g, B, R, heads * hd), normal(g, kv, prefix + 9, hd), normal(g, kv, prefix + 9, hd)
    k, v = normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    pk[:, prefix:], pv[:, prefix:] = wrong, wrong
    for b in range(B):
        k[b, :, starts[b] + counts[b]:], v[b, :, starts[b] + counts[b]:] = wrong, wrong
    k[0, :, 1, hd // 2] = wrong
    v[1, :, starts[1] + 2, 1] = wrong
    k[2, :, starts[2] + 2], v[2, :, starts[2] + 1] = wrong, wrong
    q[3, 1] = float("nan")
    fine = torch.zeros(B, R, dtype=torch.bool, device="cuda")
    for b, r in ((0, 0), (1, 0), (1, 1), (2, 0), (3, 0), (4, 0)):
        fine[b, r] = True
    got = run_attention(kc, q, pk, pv, prefix, k, v, starts, counts, heads, kv, hd)
    want, top = attention_64(q, pk, pv, prefix, k, v, starts, [1, 2, 1, 1, 1], heads, kv, hd, got)
    close(got[fine], want[fine], hd, top)
    assert not got[1, 2].isfinite().all() and not got[2, 1].isfinite().all() and not got[3, 1].isfinite().any()
    assert (got[3, 2] == -7.0).all() and (got[4, 1:] == -7.0).all()


@pytest.mark.parametrize("hd,gs", [(128, 64), (64, 64), (64, 16), (128, 128), (96, 32)])
def test_shared_attention_quantizes_its_output(kc, hd, gs):
    heads, kv, B, R, prefix, S = 8, 2, 3, 2, 100, 40
    g = generator(7)
    args = (1.5 * normal(g, B, R, heads * hd), normal(g, kv, prefix, hd), normal(g, kv, prefix, hd), prefix,
            normal(g, B, kv, S, hd), normal(g, B, kv, S, hd), [10, 20, 38], [2, 0, 1], heads, kv, hd)
    out, oq, os_ = run_attention(kc, *args, gs=gs)
    assert torch.equal(out, run_attention(kc, *args))
    wq, ws = kc.quantize(out, gs)
    for b, n in ((0, 2), (2, 1)):
        assert torch.equal(oq[b, :n], wq[b, :n]) and torch.equal(os_[b, :n], ws[b, :n])
    assert (oq[1] == 99).all() and (oq[2, 1:] == 99).all() and (os_[1] == -1).all() and (os_[2, 1:] == -1).all()


@pytest.mark.parametrize("starts,counts", [([0, -1, 0], [1, 1, 1]), ([0, 40, 0], [1, 1, 1]), ([0, 39, 0], [1, 2, 1]),
                                           ([0, 0, 0], [1, 3, 1]), ([0, 0, 0], [1, -1, 1]),
                                           ([0, 2 ** 31 - 1, 0], [1, 2, 1])])
def test_shared_attention_reports_bad_requests(kc, starts, counts):
    heads, kv, hd, B, R, prefix, S = 4, 2, 64, 3, 2, 50, 40
    g = generator(8)
    q, pk, pv = normal(g, B, R, heads * hd), normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    out = torch.full_like(q, -7.0)
    with pytest.raises(kc.KernelError, match="rejected its arguments"):
        run_attention(kc, q, pk, pv, prefix, k, v, starts, counts, heads, kv, hd, out=out)
    assert (out[1] == -7.0).all()
    want, top = attention_64(q, pk, pv, prefix, k, v, [0, 0, 0], [1, 0, 1], heads, kv, hd, torch.full_like(q, -7.0))
    close(out, want, hd, top)


@pytest.mark.parametrize("batch,rows,heads,kv,hd,prefix,room", [(700, 1, 8, 8, 64, 70, 40), (300, 3, 16, 8, 64, 333, 700),
                                                                 (260, 2, 6, 2, 128, 0, 150)])
def test_shared_attention_many_requests(kc, batch, rows, heads, kv, hd, prefix, room):
    """Many more items than CTAs: requests of all lengths, a third of them out of use, partly used rows."""
    g = generator(batch)
    q = normal(g, batch, rows, heads * hd)
    pk, pv = normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, batch, kv, room, hd), normal(g, batch, kv, room, hd)
    counts = torch.randint(-rows, rows + 1, (batch,), device="cuda", generator=g).clamp(min=0)
    starts = (torch.rand(batch, device="cuda", generator=g) * (room - rows)).long()
    got = run_attention(kc, q, pk if prefix else None, pv if prefix else None, prefix, k, v, starts.tolist(),
                        counts.tolist(), heads, kv, hd)
    row = torch.arange(rows, device="cuda")
    q64 = q.double().view(batch, rows, kv, heads // kv, hd)
    s = torch.cat([torch.einsum("brkgd,kpd->brkgp", q64, pk.double()), torch.einsum("brkgd,bkpd->brkgp", q64, k.double())],
                  -1) / hd ** 0.5
    seen = torch.arange(room, device="cuda") <= (starts[:, None] + row)[..., None]
    seen = torch.cat([torch.ones(batch, rows, prefix, dtype=torch.bool, device="cuda"), seen], -1)
    top = float(s.abs().max())
    w = s.masked_fill(~seen[:, :, None, None], float("-inf")).softmax(-1)
    want = torch.einsum("brkgp,kpd->brkgd", w[..., :prefix], pv.double()) + \
        torch.einsum("brkgp,bkpd->brkgd", w[..., prefix:], v.double())
    used = row < counts[:, None]
    close(got[used], want.reshape(batch, rows, -1)[used], hd, top)
    assert (got[~used] == -7.0).all()


@pytest.mark.parametrize("hd,batch,rows,prefix,room", [(64, 1, 2, 150000, 40), (128, 3, 1, 20, 70000), (128, 512, 4, 2085, 64)])
def test_shared_attention_long_splits(kc, hd, batch, rows, prefix, room):
    """More positions than the splits hold in one run of the accumulators: by the number of splits, and by the work's size
    for many rows."""
    heads, kv = (64, 2) if batch > 100 else (4, 2)
    g = generator(hd + batch)
    q = normal(g, batch, rows, heads * hd)
    pk, pv = normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, batch, kv, room, hd), normal(g, batch, kv, room, hd)
    starts = [(room - rows) * (b + 1) // batch for b in range(batch)]
    got = run_attention(kc, q, pk, pv, prefix, k, v, starts, [rows] * batch, heads, kv, hd)
    some = sorted({0, batch // 2, batch - 1})
    want, top = attention_64(q[some], pk, pv, prefix, k[some], v[some], [starts[b] for b in some], [rows] * len(some),
                             heads, kv, hd, got[some])
    close(got[some], want, hd, top)


# Root mean square, relative, of results in which no score's error shows: the tensor cores cut a tile's product four times
# by up to 2^-23 of what has come together by then (5/8 of it on average over the four), a probability and a value are
# pairs of half-precision numbers (2^-23 at most each), and the sums over tiles and splits, the weights' sum, the joins
# and the division are some 50 roundings of 2^-24 at most: random ones, of 2^-24 sqrt(50 / 3) together.
PRODUCTS = (4 * 5 / 8 + 2) * 2.0 ** -23 + 4 * 2.0 ** -24


def norm_error(got, want):
    return float((got.double() - want).norm() / want.norm())


LONG = [(64, 1, 2, 150000, 40), (128, 3, 1, 20, 70000), (128, 512, 4, 2085, 64), (128, 8, 1, 2048, 40), (64, 64, 4, 1024, 30)]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c)))
def test_shared_attention_of_equal_values_is_the_value(kc, case):
    """Whatever the weights, and however many tiles a split has."""
    hd, batch, rows, prefix, room = case
    heads, kv = (32, 2) if batch > 2 else (4, 2)
    g = generator(hd + batch + 1)
    q, pk, k = normal(g, batch, rows, heads * hd), normal(g, kv, prefix, hd), normal(g, batch, kv, room, hd)
    value = normal(g, kv, 1, hd)
    pv, v = value.expand(kv, prefix, hd).contiguous(), value.expand(batch, kv, room, hd).contiguous()
    got = run_attention(kc, q, pk, pv, prefix, k, v, [room - rows] * batch, [rows] * batch, heads, kv, hd)
    want = value.double().expand(kv, heads // kv, hd).reshape(-1)
    assert norm_error(got, want.expand_as(got)) <= PRODUCTS


@pytest.mark.parametrize("place", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(map(str, c)))
def test_shared_attention_of_one_dominant_position(kc, case, place):
    """A position with 0.998 of the weight, at the start, in the middle and at the end of the prefix: its value is the
    result, with no part of it lost or added on the way."""
    hd, batch, rows, prefix, room = case
    heads, kv = (32, 2) if batch > 2 else (4, 2)
    g = generator(hd + batch + 2)
    q = torch.ones(batch, rows, heads * hd, device="cuda")
    pk, pv = normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, batch, kv, room, hd), normal(g, batch, kv, room, hd)
    pk[:, int(place * (prefix - 1))] = (0.5 + float(np.log(500 * (prefix + room)))) / hd ** 0.5
    got = run_attention(kc, q, pk, pv, prefix, k, v, [room - rows] * batch, [rows] * batch, heads, kv, hd)
    some = sorted({0, batch - 1})
    want, _ = attention_64(q[some], pk, pv, prefix, k[some], v[some], [room - rows] * len(some), [rows] * len(some), heads,
                           kv, hd, got[some])
    assert norm_error(got[some], want) <= PRODUCTS


@pytest.mark.parametrize("hd", [128, 64, 96, 32, 256, 33])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e10, 1e20, 3.4e38])
def test_shared_attention_unseen_values_change_nothing(kc, hd, size):
    """Finite keys and values of any size where a row does not see them (behind its own position, behind the prefix, behind
    the request's last row) against zeros in their place: the same bits."""
    heads, kv, B, R, prefix, S = 8, 2, 3, 4, 130, 90
    starts, counts = [2, 61, 70], [4, 4, 2]
    g = generator(17)
    q, pk, pv = normal(g, B, R, heads * hd), normal(g, kv, prefix + 9, hd), normal(g, kv, prefix + 9, hd)
    k, v = normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    for row in range(3):
        outs = []
        for factor in (0.0, size):
            a = [t.clone() for t in (pk, pv, k, v)]
            for t, sign in zip(a[:2], (1, -1)):
                t[:, prefix:] = t[:, prefix:].sign() * sign * factor
            for t, sign in zip(a[2:], (-1, 1)):
                for b in range(B):
                    t[b, :, starts[b] + row + 1:] = t[b, :, starts[b] + row + 1:].sign() * sign * factor
            outs.append(run_attention(kc, q, a[0], a[1], prefix, a[2], a[3], starts, counts, heads, kv, hd))
        assert torch.equal(outs[0][:, :row + 1], outs[1][:, :row + 1])


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1e8, 1e12])
def test_shared_attention_large_values_of_no_weight(kc, hd, size):
    """Positions with next to no weight (e^-60 and less) whose values are larger than the others' by `size`, and one whose
    key is: they cost the others nothing. Scores of the positions that count are below 6, so that a weight is off by
    2^-24 (6 sqrt(head_dim) + 8) of itself."""
    heads, kv, B, R, prefix, S = 8, 2, 2, 2, 1000, 70
    g = generator(18)
    q = 0.7 * normal(g, B, R, heads * hd)
    q.view(B, R, heads, hd)[..., 0] = 4.0
    pk, pv = normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    pk[..., 0], k[..., 0] = 0.0, 0.0
    for t in (5, 333, 340, 999):
        pk[:, t, 0], pv[:, t] = -20 * hd ** 0.5, size * pv[:, t]
    k[0, :, 3, 0], v[0, :, 3] = -20 * hd ** 0.5, size * v[0, :, 3]
    pk[:, 777] *= 0.0
    pk[:, 777, 0] = -20 * hd ** 0.5 * size
    got = run_attention(kc, q, pk, pv, prefix, k, v, [S - R, 40], [R] * B, heads, kv, hd)
    want, _ = attention_64(q, pk, pv, prefix, k, v, [S - R, 40], [R] * B, heads, kv, hd, got)
    assert norm_error(got, want) <= U * (6 * hd ** 0.5 + 8)


@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("size", [1e-28, 1e-15, 1e15, 1e26])
def test_shared_attention_keys_and_values_of_any_power(kc, hd, size):
    """Each position's key of a power of its own between 1 / 1000 and 1000 times `size`, queries the other way; values of
    powers 2^-40 to 2^40, those of the largest weighing most."""
    heads, kv, B, R, prefix, S = 8, 2, 3, 2, 500, 130
    g = generator(20)
    power = lambda *shape: 2.0 ** torch.randint(-10, 11, shape, device="cuda", generator=g)  # noqa: E731
    q = normal(g, B, R, heads * hd) / (1000 * size)
    pk, k = normal(g, kv, prefix, hd) * power(kv, prefix, 1) * size, normal(g, B, kv, S, hd) * power(B, kv, S, 1) * size
    wide = lambda *shape: 2.0 ** torch.randint(-40, 41, shape, device="cuda", generator=g)  # noqa: E731
    pv, v = normal(g, kv, prefix, hd) * wide(kv, prefix, 1), normal(g, B, kv, S, hd) * wide(B, kv, S, 1)
    starts = [S - R, 64, 3]
    got = run_attention(kc, q, pk, pv, prefix, k, v, starts, [R] * B, heads, kv, hd)
    want, top = attention_64(q, pk, pv, prefix, k, v, starts, [R] * B, heads, kv, hd, got)
    assert norm_error(got, want) <= U * (top * hd ** 0.5 + 8)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1e9, 1e15])
def test_shared_attention_large_scores(kc, hd, size):
    """Scores so far apart that one position has all the weight, values of any power."""
    heads, kv, B, R, prefix, S = 8, 2, 3, 2, 700, 66
    g = generator(19)
    q = size * normal(g, B, R, heads * hd).sign()
    signs = normal(g, kv, prefix, hd).sign()
    pk, pv = signs * 1e-4, normal(g, kv, prefix, hd) * 2.0 ** torch.randint(-30, 31, (kv, prefix, 1), device="cuda", generator=g)
    k, v = 1e-4 * normal(g, B, kv, S, hd).sign(), normal(g, B, kv, S, hd)
    best = torch.randint(0, prefix, (B, R, heads), device="cuda", generator=g)
    for b in range(B):
        for r in range(R):
            for h in range(heads):
                pk[h // (heads // kv), best[b, r, h]] = 1000 * q[b, r, h * hd:(h + 1) * hd].sign()
    got = run_attention(kc, q, pk, pv, prefix, k, v, [S - R] * B, [R] * B, heads, kv, hd)
    want, _ = attention_64(q, pk, pv, prefix, k, v, [S - R] * B, [R] * B, heads, kv, hd, got)
    got, want = got.view(B, R, heads, hd), want.view(B, R, heads, hd)
    # Where the two largest scores are nearer than head_dim roundings, the roundings decide.
    top = torch.einsum("brkgd,kpd->brkgp", q.double().view(B, R, kv, heads // kv, hd), pk.double()).flatten(2, 3).topk(2).values
    clear = top[..., 0] - top[..., 1] > 8 * U * hd * top[..., 0]
    assert clear.sum() > clear.numel() / 2
    assert ((got.double() - want).abs() <= PRODUCTS * want.abs().amax(-1, keepdim=True))[clear].all()


@pytest.mark.parametrize("case", LONG + [(128, 64, 4, 8192, 64), (256, 8, 2, 700, 60), (33, 8, 2, 700, 60)],
                         ids=lambda c: "-".join(map(str, c)))
def test_shared_attention_error(kc, case):
    """The root mean square error of ordinary inputs: scores with a standard deviation of 1.5 are off by 2^-24 sqrt(head_dim)
    of that at most (head_dim roundings, random ones), which moves the weights by as much of themselves; the products'
    roundings join it."""
    hd, batch, rows, prefix, room = case
    heads, kv = (32, 2) if batch > 2 else (4, 2)
    g = generator(hd + batch + 3)
    q = 1.5 * normal(g, batch, rows, heads * hd)
    pk, pv = normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, batch, kv, room, hd), normal(g, batch, kv, room, hd)
    starts = [(room - rows) * (b + 1) // batch for b in range(batch)]
    got = run_attention(kc, q, pk, pv, prefix, k, v, starts, [rows] * batch, heads, kv, hd)
    some = sorted({0, batch // 2, batch - 1})
    want, _ = attention_64(q[some], pk, pv, prefix, k[some], v[some], [starts[b] for b in some], [rows] * len(some), heads,
                           kv, hd, got[some])
    assert norm_error(got[some], want) <= PRODUCTS + U * 1.5 * hd ** 0.5


def test_shared_attention_is_the_engines_attention(kc):
    """One request whose positions are cut into a prefix and its own: k_attention_batch_kv over the whole cache."""
    heads, kv, hd, R, prefix, S = 32, 8, 128, 4, 300, 80
    g = generator(9)
    n = prefix + S
    q, kc_, vc = 1.5 * normal(g, 1, R, heads * hd), normal(g, kv, n, hd), normal(g, kv, n, hd)
    want = torch.zeros(R, heads * hd, device="cuda")
    work = kc.attention_work(heads, kv, hd, n, rows=R)
    kc.k_attention_batch_kv(want, q, kc_, vc, work, heads, kv, hd, n, n - R, R)
    kc.status()
    kc.k_attention_free(work)
    got = run_attention(kc, q, kc_, vc, prefix, kc_[None, :, prefix:].contiguous(), vc[None, :, prefix:].contiguous(),
                        [S - R], None, heads, kv, hd)
    close(got[0], want.double(), hd, 8.0)


def test_shared_attention_offsets_past_32_bits(kc):
    """Caches of more than 2^31 values: the last head of the prefix and the last request lie behind them."""
    heads, kv, hd, B, R, prefix = 8, 8, 128, 17, 1, 70
    room, S = 2_200_000, 131_072
    g = generator(10)
    pk, pv = torch.empty(kv, room, hd, **CUDA), torch.empty(kv, room, hd, **CUDA)
    k, v = torch.empty(B, kv, S, hd, **CUDA), torch.empty(B, kv, S, hd, **CUDA)
    assert pk.numel() > 2 ** 31 and k.numel() > 2 ** 31
    q = normal(g, B, R, heads * hd)
    starts, counts = [0] * B, [0] * B
    starts[-1], counts[-1] = 90, 1
    for t in (pk, pv):
        t[:, :prefix] = normal(g, kv, prefix, hd)
    for t in (k, v):
        t[-1, :, :91] = normal(g, kv, 91, hd)
    got = run_attention(kc, q, pk, pv, prefix, k, v, starts, counts, heads, kv, hd)
    keys, values = torch.cat([pk[:, :prefix], k[-1, :, :91]], 1), torch.cat([pv[:, :prefix], v[-1, :, :91]], 1)
    want, top = attention_64(q[-1:], keys[:, :0], values[:, :0], 0, keys[None], values[None], [prefix + 90], [1], heads, kv,
                             hd, q[-1:])
    close(got[-1:], want, hd, top)


# ---- adapters ----------------------------------------------------------------------------------------------------------

LORA = [  # rows, adapters, ranks, n, d, dtype
    (1, 1, [8], 2048, 2048, torch.bfloat16),
    (1, 1, [1], 1, 1, torch.float32),
    (3, 2, [4, 16], 64, 40, torch.float16),
    (7, 3, [5, 0, 12], 100, 33, torch.bfloat16),
    (33, 5, [32, 16, 8, 32, 16], 512, 1031, torch.float32),
    (64, 64, [16] * 64, 512, 512, torch.bfloat16),
    (65, 4, [64, 64, 8, 3], 776, 520, torch.float16),
    (130, 2, [256, 100], 320, 260, torch.bfloat16),
    (300, 7, [64, 32, 16, 8, 4, 2, 1], 1024, 768, torch.bfloat16),
    (257, 3, [64, 64, 64], 4096, 264, torch.float32),
    (1000, 4, [64, 64, 64, 64], 512, 1000, torch.float16),
    (513, 2, [24, 40], 513, 515, torch.float32),
]


# Cases large enough for tiles of rows of one adapter: ragged last steps, ranks that fill no block, three weight types,
# tiles of few and of many rows, more adapters than the rows use.
LORA += [
    (400, 3, [64, 128, 100], 2056, 1100, torch.bfloat16),
    (900, 5, [16, 24, 1, 64, 48], 1000, 1300, torch.float16),
    (350, 2, [128, 65], 520, 904, torch.float32),
    (2100, 90, [32] * 90, 640, 2000, torch.bfloat16),
    (1500, 4, [20, 36, 7, 60], 1023, 777, torch.bfloat16),
    (700, 2, [64, 64], 8, 4000, torch.float32),
]


# One CTA a row, many outputs each, at ranks of one, two and half a unit of reads; a rank of more units than lanes.
LORA += [
    (700, 3, [8, 4, 16], 64, 3001, torch.bfloat16),
    (700, 3, [8, 2, 4], 64, 3001, torch.float32),
    (620, 3, [4, 3, 1], 40, 2600, torch.float16),
    (40, 2, [256, 132], 260, 300, torch.float32),
    (170, 3, [24, 12, 20], 2048, 96, torch.bfloat16),
]


# Long rows: several passes over n, with a ragged last one.
LORA += [
    (260, 2, [64, 24], 16384 + 72, 256, torch.bfloat16),
    (200, 1, [16], 3 * 16384 - 8, 264, torch.float32),
    (140, 2, [100, 128], 20001, 130, torch.float16),
]


def lora_inputs(case, order, seed=0):
    rows, count, ranks, n, d, dtype = case
    g = generator(rows + seed)
    a = [(normal(g, r, n) / n ** 0.5).to(dtype) for r in ranks]
    b = [(0.3 * normal(g, d, r)).to(dtype) for r in ranks]
    scale = [0.5 + 0.25 * i for i in range(count)]
    rng = np.random.default_rng(seed)
    index = {"runs": np.arange(rows) * count // rows, "each": np.arange(rows) % count,
             "mixed": rng.integers(-1, count, rows)}[order]
    return a, b, scale, torch.tensor(index, dtype=torch.int32, device="cuda"), g


def lora_64(x, base, index, a, b, scale):
    """The definition in 64 bits, and the tolerance per element."""
    want, size = base.double().clone(), torch.zeros_like(base, dtype=torch.float64)
    for i, (A, B) in enumerate(zip(a, b)):
        rows = (index == i).nonzero()[:, 0]
        want[rows] += scale[i] * ((x[rows].double() @ A.double().T) @ B.double().T)
        size[rows] += (4 * (x.shape[1] ** 0.5 + A.shape[0] ** 0.5 + 4)) * abs(scale[i]) * (
            (x[rows].double().abs() @ A.double().abs().T) @ B.double().abs().T)
    return want, U * (size + 2 * base.double().abs() + 2 * want.abs())


def kind(kc, dtype):
    return {torch.float32: kc.K_F32, torch.bfloat16: kc.K_BF16, torch.float16: kc.K_F16}[dtype]


@pytest.mark.parametrize("order", ["runs", "each", "mixed"])
@pytest.mark.parametrize("case", LORA, ids=lambda c: f"{c[0]}-{c[1]}-{max(c[2])}-{c[3]}-{c[4]}-{str(c[5])[6:]}")
def test_lora(kc, case, order):
    rows, count, ranks, n, d, dtype = case
    a, b, scale, index, g = lora_inputs(case, order)
    x, base = normal(g, rows, n), normal(g, rows, d)
    table = kc.lora_table(a, b, scale)
    out = torch.full((rows, d), -7.0, device="cuda")
    kc.k_lora_rows(out, d, base, d, x, n, index, table, count, kind(kc, dtype), max(ranks), n, d, rows)
    kc.status()
    want, tol = lora_64(x, base, index, a, b, scale)
    assert ((out.double() - want).abs() <= tol).all()
    again = base.clone()  # in place, and the same bits
    kc.k_lora_rows(again, d, again, d, x, n, index, table, count, kind(kc, dtype), max(ranks), n, d, rows)
    kc.status()
    assert torch.equal(again, out)
    kc.k_lora_rows(out, d, None, 0, x, n, index, table, count, kind(kc, dtype), max(ranks), n, d, rows)
    kc.status()
    want, tol = lora_64(x, torch.zeros_like(base), index, a, b, scale)
    assert ((out.double() - want).abs() <= tol).all()


def two_parts(x):
    """To 16 bits, as two bfloat16 numbers hold it."""
    high = x.bfloat16().double()
    return high + (x.double() - high).bfloat16().double()


@pytest.mark.parametrize("order", ["runs", "each"])
@pytest.mark.parametrize("case", LORA, ids=lambda c: f"{c[0]}-{c[1]}-{max(c[2])}-{c[3]}-{c[4]}-{str(c[5])[6:]}")
def test_lora_error(kc, case, order):
    """The root mean square error of the products alone. The tensor cores cut a sum by half a step (0.36 * 2^-23 on average
    over its mantissas) of what it has come to, 2/3 of its end on average over a random run: once for every 48 elements
    of a CTA's eighth of n (16384 a launch at most), and in the second product for every 16 ranks and eight small terms.
    Some dozen random roundings, 2^-24 sqrt(12 / 3), join it. Activations and vectors of 16 bits would not pass."""
    rows, count, ranks, n, d, dtype = case
    a, b, scale, index, g = lora_inputs(case, order, 2)
    x = normal(g, rows, n)
    out = torch.full((rows, d), -7.0, device="cuda")
    kc.k_lora_rows(out, d, None, 0, x, n, index, kc.lora_table(a, b, scale), count, kind(kc, dtype), max(ranks), n, d, rows)
    kc.status()
    want, _ = lora_64(x, torch.zeros(rows, d, device="cuda"), index, a, b, scale)
    cuts = min(n, 16384) / 8 / 48 + max(ranks) / 16 + 8
    bound = cuts * 0.36 * 2 / 3 * 2.0 ** -23 + 2 * U
    assert norm_error(out, want) <= bound
    if 64 <= n <= 4096 and rows * d > 1000:
        less = torch.zeros_like(want)
        for i, (A, B) in enumerate(zip(a, b)):
            at = (index == i).nonzero()[:, 0]
            h = two_parts(two_parts(x[at]) @ A.double().T)
            less[at] = scale[i] * (h @ B.double().T)
        assert norm_error(less, want) > bound


@pytest.mark.parametrize("rows", [5, 200, 3000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lora_strides_and_alignment(kc, rows, dtype):
    """Rows inside wider buffers (their gaps stay as they were), matrices at odd addresses."""
    n, d, ranks = (264, 130, [16, 24]) if rows < 1000 else (808, 334, [16, 24])
    a, b, scale, index, g = lora_inputs((rows, 2, ranks, n, d, dtype), "mixed")
    x, base = normal(g, rows, n + 5), normal(g, rows, d + 3)
    out = torch.full((rows, d + 7), -7.0, device="cuda")
    shift = lambda m: torch.cat([m.new_zeros(1), m.reshape(-1)])[1:].view(m.shape)  # noqa: E731
    for am, bm, x0 in ((a, b, 0), ([shift(m) for m in a], [shift(m) for m in b], 1)):
        table = kc.lora_table(am, bm, scale)
        kc.k_lora_rows(out, d + 7, base, d + 3, x.view(-1)[x0:], n + 5, index, table, 2, kind(kc, dtype), 24, n, d, rows)
        kc.status()
        want, tol = lora_64(x.view(-1)[x0:].as_strided((rows, n), (n + 5, 1)), base[:, :d].contiguous(), index, a, b,
                            scale)
        assert ((out[:, :d].double() - want).abs() <= tol).all()
        assert (out[:, d:] == -7.0).all()


@pytest.mark.parametrize("rows", [6, 150, 4000])
def test_lora_reports_bad_rows(kc, rows):
    n, d = (64, 72) if rows < 1000 else (1024, 520)
    a, b, scale, index, g = lora_inputs((rows, 2, [8, 16], n, d, torch.bfloat16), "each")
    x, base = normal(g, rows, n), normal(g, rows, d)
    table = kc.lora_table(a, b, scale)
    for bad, max_rank in ((2, 16), (-2, 16), (2 ** 31 - 1, 16), (1, 8)):
        idx = torch.zeros_like(index)
        idx[3] = bad
        out = torch.full((rows, d), -7.0, device="cuda")
        kc.k_lora_rows(out, d, base, d, x, n, idx, table, 2, kc.K_BF16, max_rank, n, d, rows)
        with pytest.raises(kc.KernelError, match="rejected its arguments"):
            kc.status()
        want, tol = lora_64(x, base, torch.where(torch.arange(rows, device="cuda") == 3, -1, idx), a, b, scale)
        assert ((out.double() - want).abs() <= tol).all()
        assert torch.equal(out[3], base[3])


@pytest.mark.parametrize("rows", [4, 150, 4000])
def test_lora_nonfinite_rows_stay_their_own(kc, rows):
    """An infinity or NaN in one row, or in an adapter, shows in the rows that use it and in no other."""
    n, d = (128, 64) if rows < 1000 else (2048, 512)
    a, b, scale, index, g = lora_inputs((rows, 3, [8, 8, 8], n, d, torch.bfloat16), "each")
    x, base = normal(g, rows, n), normal(g, rows, d)
    x[1, 5] = float("inf")
    a[2][:] = float("nan")
    out = torch.empty(rows, d, device="cuda")
    kc.k_lora_rows(out, d, base, d, x, n, index, kc.lora_table(a, b, scale), 3, kc.K_BF16, 8, n, d, rows)
    kc.status()
    sick = (index == 2) | (torch.arange(rows, device="cuda") == 1)
    assert not out[sick].isfinite().any() and out[~sick].isfinite().all()


@pytest.mark.parametrize("rows", [4, 150, 4000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lora_rows_of_any_numbers(kc, rows, dtype):
    """Activations up to the largest finite ones, whose results are finite, and infinities, whose results are infinities or
    NaN as the formula gives them, whichever kernel runs."""
    n, d, ranks = (128, 64, [1, 8, 3]) if rows < 1000 else (2048, 512, [1, 8, 3])
    a, b, scale, index, g = lora_inputs((rows, 3, ranks, n, d, dtype), "each", 3)
    x, base = normal(g, rows, n), normal(g, rows, d)
    for m in a:
        m[:, 7] = m[:, 7].sign() * 2.0 ** -20
        m[:, 8] = m[:, 8].sign() * 2.0 ** -24
    huge = torch.finfo(torch.float32).max
    for r in range(0, rows, 31):  # of each adapter in turn
        x[r, 5] = float("inf")
    for r in range(1, rows, 31):
        x[r, 7] = huge
    for r in range(2, rows, 31):
        x[r, 7], x[r, 8] = -huge, 3.4e38
    for r in range(3, rows, 31):
        x[r, 5], x[r, 6] = float("inf"), float("-inf")
    out = torch.empty(rows, d, device="cuda")
    kc.k_lora_rows(out, d, base, d, x, n, index, kc.lora_table(a, b, scale), 3, kind(kc, dtype), 8, n, d, rows)
    kc.status()
    want, tol = lora_64(x, base, index, a, b, scale)
    finite = want.isfinite()
    assert finite[1::31].all() and not finite[0::31].any() and want[0::31].isinf().any()
    assert ((out.double() - want).abs() <= tol)[finite].all()
    assert torch.equal(out[~finite].isnan(), want[~finite].isnan())
    inf = want.isinf()
    assert torch.equal(out[inf].double(), want[inf])


@pytest.mark.parametrize("n", [1024, 16384 + 72])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lora_rows_of_any_numbers_in_place(kc, n, dtype):
    """Rows that are not finite, over one launch and over two parts of n, with base as the output: the same bits as beside
    it, and every row's own result."""
    rows, d, ranks = 700, 300, [16, 5, 128]
    a, b, scale, index, g = lora_inputs((rows, 3, ranks, n, d, dtype), "mixed", 4)
    x, base = normal(g, rows, n), normal(g, rows, d)
    sick = torch.arange(0, rows, 23, device="cuda")
    x[sick, torch.randint(0, n, (len(sick),), device="cuda", generator=g)] = float("inf")
    x[sick[::2], n - 1] = float("nan")
    table = kc.lora_table(a, b, scale)
    out, again = torch.full((rows, d), -7.0, device="cuda"), base.clone()
    kc.k_lora_rows(out, d, base, d, x, n, index, table, 3, kind(kc, dtype), 128, n, d, rows)
    kc.k_lora_rows(again, d, again, d, x, n, index, table, 3, kind(kc, dtype), 128, n, d, rows)
    kc.status()
    assert torch.equal(out.isfinite(), again.isfinite())
    assert torch.equal(out[out.isfinite()], again[out.isfinite()])
    want, tol = lora_64(x, base, index, a, b, scale)
    finite = want.isfinite()
    assert torch.equal(out.isfinite(), finite) and ((out.double() - want).abs() <= tol)[finite].all()
    with_adapter = sick[index[sick] >= 0]
    assert len(with_adapter) > 10 and not out[with_adapter].isfinite().any()


def test_lora_more_rows_than_a_launch_takes(kc):
    """Over 16384 rows: several launches, each with its own part of the index."""
    case = (20000, 3, [16, 8, 24], 256, 264, torch.bfloat16)
    rows, count, ranks, n, d, dtype = case
    a, b, scale, index, g = lora_inputs(case, "mixed")
    x, base = normal(g, rows, n), normal(g, rows, d)
    out = torch.full((rows, d), -7.0, device="cuda")
    kc.k_lora_rows(out, d, base, d, x, n, index, kc.lora_table(a, b, scale), count, kc.K_BF16, 24, n, d, rows)
    kc.status()
    want, tol = lora_64(x, base, index, a, b, scale)
    assert ((out.double() - want).abs() <= tol).all()


# ---- drafts ------------------------------------------------------------------------------------------------------------

def verify_64(target, draft, drafted, counts, uniforms, temperature, vocab):
    """Request by request, in 64 bits: (accepted, tokens)."""
    B, R = drafted.shape
    accepted, tokens = np.full(B, -9), np.full((B, R + 1), -9)
    for b in range(B):
        if counts[b] < 0:
            continue
        tokens[b] = -1
        t = float(temperature[b])

        def softmax(row):
            x = row[:vocab].astype(np.float64) / t
            e = np.exp(x - x.max())
            return e / e.sum()

        for j in range(counts[b] + 1):
            row = target[b, j, :vocab]
            x = drafted[b, j] if j < counts[b] else -1
            if t == 0:
                last = int(np.argmax(row))
                if last == x:
                    tokens[b, j] = x
                    continue
            else:
                w = softmax(row)
                if j < counts[b]:
                    q = softmax(draft[b, j]) if draft is not None else (np.arange(vocab) == x).astype(np.float64)
                    if float(uniforms[b, j]) * q[x] < w[x]:
                        tokens[b, j] = x
                        continue
                    w = np.maximum(w - q, 0)
                run = np.cumsum(w)
                last = int(np.argmax(run > float(uniforms[b, R]) * run[-1])) if run[-1] > 0 else int(np.argmax(row))
            tokens[b, j] = last
            accepted[b] = j
            break
    return accepted, tokens


def run_verify(kc, target, draft, drafted, counts, uniforms, temperature, vocab, rows):
    B = target.shape[0]
    dev = lambda x, t: None if x is None else torch.tensor(np.asarray(x), dtype=t, device="cuda")  # noqa: E731
    accepted = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    tokens = torch.full((B, rows + 1), -9, dtype=torch.int32, device="cuda")
    work = torch.empty(kc.k_verify_bytes(vocab, B, rows), dtype=torch.uint8, device="cuda")
    tg, dr = dev(target, torch.float32), dev(draft, torch.float32)
    kc.k_verify_draft(accepted, tokens, tg, target.shape[2], dr, 0 if draft is None else draft.shape[2],
                      dev(drafted, torch.int32), dev(counts, torch.int32), dev(uniforms, torch.float32),
                      dev(temperature, torch.float32), vocab, B, rows, work)
    kc.status()
    return accepted.cpu().numpy(), tokens.cpu().numpy()


def verify_inputs(B, R, vocab, ld, drafts, seed, spread=3.0):
    rng = np.random.default_rng(seed)
    target = (spread * rng.standard_normal((B, R + 1, ld))).astype(np.float32)
    draft = (target[:, :R] + 0.7 * rng.standard_normal((B, R, ld))).astype(np.float32)
    temperature = np.where(rng.random(B) < 0.25, 0, 0.5 + rng.random(B)).astype(np.float32)
    temperature[0] = 0.8
    noisy = draft[:, :, :vocab] / np.maximum(temperature, 0.01)[:, None, None] + rng.gumbel(size=(B, R, vocab))
    drafted = noisy.argmax(-1).astype(np.int32) if R else np.zeros((B, 0), np.int32)
    counts = rng.integers(-1, R + 1, B)
    counts[0] = R
    if R and B > 2:
        drafted[2] = target[2, :R, :vocab].argmax(-1)  # drafts a greedy request accepts
        temperature[2], counts[2] = 0, R
    uniforms = rng.random((B, R + 1), dtype=np.float32)
    return target, draft if drafts else None, drafted, counts, uniforms, temperature


VERIFY = [(1, 0, 1, 1), (1, 1, 2, 2), (2, 1, 7, 9), (5, 4, 129, 129), (9, 3, 1000, 1000), (3, 8, 4097, 4100),
          (17, 5, 32000, 32001), (4, 2, 128256, 128256), (3, 64, 300, 300), (70, 1, 513, 515)]


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("case", VERIFY, ids=lambda c: "-".join(map(str, c)))
def test_verify(kc, case, drafts):
    B, R, vocab, ld = case
    for seed in range(3):
        args = verify_inputs(B, R, vocab, ld, drafts, seed + 10 * B)
        want = verify_64(*args, vocab)
        got = run_verify(kc, *args, vocab, R)
        assert (got[0] == want[0]).all() and (got[1] == want[1]).all()


def test_verify_draws_follow_the_distribution(kc):
    """One row at many numbers: the chosen token is where the running sum passes each of them."""
    vocab, B = 5003, 512
    rng = np.random.default_rng(4)
    target = np.repeat((3 * rng.standard_normal((1, 1, vocab))).astype(np.float32), B, 0)
    uniforms = np.linspace(0, 1, B, endpoint=False, dtype=np.float32)[:, None]
    uniforms[-1] = np.nextafter(np.float32(1), np.float32(0))
    args = (target, None, np.zeros((B, 0), np.int32), None, uniforms, np.ones(B, np.float32))
    want = verify_64(*args[:3], np.zeros(B, int), *args[4:], vocab)
    got = run_verify(kc, *args, vocab, 0)
    assert (got[1] == want[1]).all() and (got[0] == 0).all()


def test_verify_edges(kc):
    """Masked vocabularies, ties, a draft equal to the target, certain and impossible drafts."""
    vocab, R = 600, 2
    rng = np.random.default_rng(5)
    low, inf = np.finfo(np.float32).min, np.float32(np.inf)
    row = rng.standard_normal(vocab).astype(np.float32)
    masked, lowest, one, tied, same = row.copy(), row.copy(), np.full(vocab, -inf), np.zeros(vocab), row.copy()
    masked[:500], lowest[100:] = -inf, low
    one[77] = -3.0
    tied[5::7] = 2.0
    negzero = np.full(vocab, -1.0)
    negzero[40], negzero[41] = -0.0, 0.0
    rows = [masked, lowest, one, tied, same, negzero, np.full(vocab, low)]
    target = np.stack([np.stack([r, r, r]) for r in rows for _ in range(4)]).astype(np.float32)
    B = len(target)
    draft = target[:, :R].copy()
    drafted = rng.integers(0, vocab, (B, R)).astype(np.int32)
    drafted[:, 0] = target[:, 0].argmax(-1)
    drafted[1::4] = 550
    draft[2::4] = rng.standard_normal((len(draft[2::4]), R, vocab))
    uniforms = rng.random((B, R + 1), dtype=np.float32)
    uniforms[::3, :R] = np.nextafter(np.float32(1), np.float32(0))
    uniforms[1::3, R] = 0.0
    temperature = np.where(np.arange(B) % 4 == 3, 0, 1).astype(np.float32)
    for d in (draft, None):
        args = (target, d, drafted, np.full(B, R), uniforms, temperature)
        want = verify_64(*args, vocab)
        got = run_verify(kc, *args, vocab, R)
        for b in range(B):  # a draft of probability zero under draft and target leaves no residual to draw from
            assert got[0][b] == want[0][b], b
            assert (got[1][b] == want[1][b]).all(), b


def test_verify_tiny_and_huge_temperatures(kc):
    vocab, R = 257, 1
    rng = np.random.default_rng(6)
    target = rng.standard_normal((4, 2, vocab)).astype(np.float32)
    args = (target, None, target[:, :1].argmax(-1).astype(np.int32), np.ones(4, int), rng.random((4, 2), dtype=np.float32),
            np.array([1e-30, 1e-3, 1e6, 1e30], np.float32))
    want = verify_64(*args, vocab)
    got = run_verify(kc, *args, vocab, R)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("top,t", [(20.0, 1e-8), (1500.0, 1e-6), (9.0, 1e-9), (17.0, 1.4e-9), (-20.0, 1e-8), (1e4, 3e-5),
                                   (300.0, 2e-7)])
def test_verify_low_temperatures(kc, top, t, drafts):
    """Temperatures whose 700-fold is about a step of the largest logit: neighbouring numbers, ties and all the others
    far below."""
    vocab, B, R = 4200, 6, 2
    rng = np.random.default_rng(15)
    target = (top - 1.0 - abs(rng.standard_normal((B, R + 1, vocab)))).astype(np.float32)
    top = np.float32(top)
    target[:, :, 1234] = top
    target[1::2, :, 4100] = top  # a tie
    target[2::3, :, 77] = np.nextafter(top, np.float32(-np.inf))
    draft = target[:, :R] - (rng.random((B, R, vocab)) < 0.5).astype(np.float32)
    drafted = np.full((B, R), 1234, np.int32)
    drafted[3:, 1] = [4100, 500, 77]
    uniforms = rng.random((B, R + 1), dtype=np.float32)
    args = (target, draft if drafts else None, drafted, np.full(B, R), uniforms, np.full(B, t, np.float32))
    want = verify_64(*args, vocab)
    got = run_verify(kc, *args, vocab, R)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()


@pytest.mark.parametrize("what", ["nan", "inf", "empty", "draft_nan", "token", "negative", "count", "cold", "temp_nan"])
def test_verify_reports(kc, what):
    """A needed row without a distribution, or arguments that mean nothing: no answer for that request, others whole."""
    B, R, vocab = 3, 2, 700
    target, draft, drafted, counts, uniforms, temperature = verify_inputs(B, R, vocab, vocab, True, 7)
    counts[:], temperature[:] = R, 1.0
    uniforms[:, :R] = 0.0  # every draft is accepted
    whole = run_verify(kc, target, draft, drafted, counts, uniforms, temperature, vocab, R)
    bad = {"nan": lambda: target.__setitem__((1, 2, 3), np.nan), "inf": lambda: target.__setitem__((1, 0, 3), np.inf),
           "empty": lambda: target.__setitem__((1, 1), -np.inf), "draft_nan": lambda: draft.__setitem__((1, 0, 9), np.nan),
           "token": lambda: drafted.__setitem__((1, 0), vocab), "negative": lambda: drafted.__setitem__((1, 1), -1),
           "count": lambda: counts.__setitem__(1, R + 1), "cold": lambda: temperature.__setitem__(1, -1.0),
           "temp_nan": lambda: temperature.__setitem__(1, np.nan)}[what]
    bad()
    dev = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device="cuda")  # noqa: E731
    accepted = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    tokens = torch.full((B, R + 1), -9, dtype=torch.int32, device="cuda")
    work = torch.empty(kc.k_verify_bytes(vocab, B, R), dtype=torch.uint8, device="cuda")
    kc.k_verify_draft(accepted, tokens, dev(target, torch.float32), vocab, dev(draft, torch.float32), vocab,
                      dev(drafted, torch.int32), dev(counts, torch.int32), dev(uniforms, torch.float32),
                      dev(temperature, torch.float32), vocab, B, R, work)
    with pytest.raises(kc.KernelError):
        kc.status()
    accepted, tokens = accepted.cpu().numpy(), tokens.cpu().numpy()
    assert accepted[1] == -1 and (tokens[1] == -1).all()
    for b in (0, 2):
        assert accepted[b] == whole[0][b] and (tokens[b] == whole[1][b]).all()


@pytest.mark.parametrize("count", [-2, -100, -2 ** 31])
def test_verify_reports_counts_below_the_unused_ones(kc, count):
    """Only -1 is a slot that is not in use; a count below it is as wrong as one above the rows."""
    B, R, vocab = 3, 2, 700
    target, draft, drafted, counts, uniforms, temperature = verify_inputs(B, R, vocab, vocab, True, 16)
    dev = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device="cuda")  # noqa: E731
    accepted = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    tokens = torch.full((B, R + 1), -9, dtype=torch.int32, device="cuda")
    work = torch.empty(kc.k_verify_bytes(vocab, B, R), dtype=torch.uint8, device="cuda")
    kc.k_verify_draft(accepted, tokens, dev(target, torch.float32), vocab, dev(draft, torch.float32), vocab,
                      dev(drafted, torch.int32), dev([R, count, -1], torch.int32), dev(uniforms, torch.float32),
                      dev(temperature, torch.float32), vocab, B, R, work)
    with pytest.raises(kc.KernelError, match="rejected its arguments"):
        kc.status()
    want = verify_64(target, draft, drafted, [R, -1, -1], uniforms, temperature, vocab)
    assert accepted.tolist() == [want[0][0], -1, -9]
    assert tokens[0].tolist() == want[1][0].tolist() and (tokens[1] == -1).all() and (tokens[2] == -9).all()


def test_verify_looks_at_no_row_behind_the_refused_draft(kc):
    B, R, vocab = 1, 3, 500
    target, draft, drafted, counts, uniforms, temperature = verify_inputs(B, R, vocab, vocab, True, 8)
    counts[:] = R
    drafted[0, 0] = target[0, 0].argmin()
    uniforms[0, 0] = 0.999
    draft[0, 0, drafted[0, 0]] = 9.0
    want = run_verify(kc, target, draft, drafted, counts, uniforms, temperature, vocab, R)
    target[0, 1:], draft[0, 1:], drafted[0, 1:] = np.nan, np.inf, -5
    got = run_verify(kc, target, draft, drafted, counts, uniforms, temperature, vocab, R)
    assert want[0][0] == 0 and (got[0] == want[0]).all() and (got[1] == want[1]).all()


# ---- together, streams and graphs --------------------------------------------------------------------------------------

def test_a_step_of_three_requests(kc):
    """One layer's attention block of a decoding step, as a batch of requests over one prompt would run it: the shared
    Q, K and V products with each request's adapters, RoPE and the K/V store into the requests' caches, attention with
    its quantized output, the output product, the classifier and the verification of the drafts. Each operator is held
    against its 64-bit form on what the operators before it gave."""
    heads, kv, hd, B, R, prefix, S, vocab, gs = 8, 2, 64, 3, 3, 150, 24, 1000, 64
    dim, dkv, rows = heads * hd, kv * hd, B * R
    g = generator(11)

    def weight(n, k):
        return kc.quantize(0.05 * normal(g, n, k), gs)

    wq, wk, wv, wo, wc = weight(dim, dim), weight(dkv, dim), weight(dkv, dim), weight(dim, dim), weight(vocab, dim)
    x = normal(g, rows, dim)
    pk, pv = normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    starts = [0, 5, 20]
    index = torch.tensor([0] * R + [-1] * R + [1] * R, dtype=torch.int32, device="cuda")
    xq, xs = kc.quantize(x, gs)
    deq = lambda q, s: (q.double().view(*s.shape, -1) * s.double()[..., None]).reshape(q.shape)  # noqa: E731
    outs = []
    for w, d in ((wq, dim), (wk, dkv), (wv, dkv)):
        out = torch.empty(rows, d, device="cuda")
        kc.k_gemm_q8(xq, xs, rows, dim, gs, [kc.segment(out, w)])
        a = [(normal(g, r, dim) / dim ** 0.5).bfloat16() for r in (16, 8)]
        b = [(0.3 * normal(g, d, r)).bfloat16() for r in (16, 8)]
        before = out.clone()
        kc.k_lora_rows(out, d, out, d, x, dim, index, kc.lora_table(a, b, [2.0, 1.0]), 2, kc.K_BF16, 16, dim, d, rows)
        kc.status()
        want, tol = lora_64(x, before, index, a, b, [2.0, 1.0])
        assert ((out.double() - want).abs() <= tol).all()
        outs.append(out)
    q, nk, nv = outs
    angles = torch.arange(prefix + S, device="cuda")[:, None] * 0.01 ** (torch.arange(0, hd, 2, device="cuda") / hd)
    cos, sin = angles.cos().repeat_interleave(2, 1), torch.stack([-angles.sin(), angles.sin()], 2).reshape(-1, hd)
    table = torch.cat([cos, sin], 1).float().contiguous()
    for b in range(B):
        at = slice(b * R, b * R + R)
        kc.k_rope_kv_store_rows(q[at], dim, nk[at], nv[at], dkv, k[b], v[b], table[prefix:], None, starts[b], R, heads,
                                kv, hd, S)
    kc.status()
    q = q.view(B, R, dim)
    out, oq, os_ = run_attention(kc, q, pk, pv, prefix, k, v, starts, None, heads, kv, hd, gs=gs)
    want, top = attention_64(q, pk, pv, prefix, k, v, starts, [R] * B, heads, kv, hd, out)
    close(out, want, hd, top)
    y = torch.empty(rows, dim, device="cuda")
    kc.k_gemm_q8(oq, os_, rows, dim, gs, [kc.segment(y, wo)])
    yq, ys = kc.quantize(y, gs)
    logits = torch.empty(rows, vocab, device="cuda")
    kc.k_gemm_q8(yq, ys, rows, dim, gs, [kc.segment(logits, wc)])
    kc.status()
    want = deq(yq, ys) @ deq(*wc).T
    assert float((logits.double() - want).norm() / want.norm()) < 1e-5
    rng = np.random.default_rng(12)
    target = 6.0 * logits.view(B, R, vocab).cpu().numpy() / float(logits.std())
    drafted = target[:, :R - 1].argmax(-1).astype(np.int32)
    args = (target.astype(np.float32), None, drafted, np.array([R - 1, 1, 0]), rng.random((B, R), dtype=np.float32),
            np.array([1.0, 0.0, 0.7], np.float32))
    want = verify_64(*args, vocab)
    got = run_verify(kc, *args, vocab, R - 1)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()


def test_captured_steps_and_side_streams(kc):
    """The three operators captured into a graph on a side stream; replays follow new inputs, starts and counts."""
    heads, kv, hd, B, R, prefix, S, vocab = 8, 2, 64, 4, 2, 100, 30, 900
    dim, rows = heads * hd, B * R
    g = generator(13)
    q, pk, pv = normal(g, B, R, dim), normal(g, kv, prefix, hd), normal(g, kv, prefix, hd)
    k, v = normal(g, B, kv, S, hd), normal(g, B, kv, S, hd)
    starts = torch.tensor([0, 3, 9, 20], dtype=torch.int32, device="cuda")
    counts = torch.tensor([2, 1, 2, 0], dtype=torch.int32, device="cuda")
    att = torch.zeros(B, R, dim, device="cuda")
    work = kc.shared_attention_work(heads, kv, hd, B, R)
    a, b, scale, index, _ = lora_inputs((rows, 2, [8, 16], dim, vocab, torch.bfloat16), "each")
    table = kc.lora_table(a, b, scale)
    logits = torch.zeros(rows, vocab, device="cuda")
    drafted = torch.randint(0, vocab, (B, R - 1), dtype=torch.int32, device="cuda", generator=g)
    uniforms = torch.rand(B, R, device="cuda", generator=g)
    temperature = torch.tensor([1.0, 0.5, 0.0, 1.0], device="cuda")
    drafts = torch.tensor([1, 0, 1, -1], dtype=torch.int32, device="cuda")
    accepted = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    tokens = torch.full((B, R), -9, dtype=torch.int32, device="cuda")
    vwork = torch.empty(kc.k_verify_bytes(vocab, B, R - 1), dtype=torch.uint8, device="cuda")

    def step():
        kc.k_attention_shared_rows(att, None, None, q, pk, pv, prefix, prefix, k, v, starts, counts, work, heads, kv, hd, S,
                                   B, R, 0)
        kc.k_lora_rows(logits, vocab, None, 0, att, dim, index, table, 2, kc.K_BF16, 16, dim, vocab, rows)
        kc.k_verify_draft(accepted, tokens, logits, vocab, None, 0, drafted, drafts, uniforms, temperature, vocab, B, R - 1,
                          vwork)

    step()
    kc.status()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        step()
    for turn in range(3):
        q.copy_(normal(g, B, R, dim))
        starts.copy_(torch.tensor([turn, 5 + turn, 1, 0], dtype=torch.int32))
        att.fill_(-7.0)
        logits.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (att, logits, accepted, tokens)]
        att.fill_(-7.0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            kc.status()
        for got, want in zip((att, logits, accepted, tokens), replayed):
            assert torch.equal(got, want)
        used = [2, 1, 2, 0]
        want, top = attention_64(q, pk, pv, prefix, k, v, starts.tolist(), used, heads, kv, hd, torch.full_like(q, -7.0))
        close(att, want, hd, top)
    kc.k_attention_free(work)


def test_two_works_on_two_streams(kc):
    """Two calls at once, each with a workspace of its own, give what each gives alone."""
    heads, kv, hd, B, R, prefix, S = 32, 8, 128, 8, 2, 2000, 64
    g = generator(14)
    sets, alone = [], []
    for _ in range(2):
        s = (normal(g, B, R, heads * hd), normal(g, kv, prefix, hd), normal(g, kv, prefix, hd), prefix,
             normal(g, B, kv, S, hd), normal(g, B, kv, S, hd), [S - R] * B, [R] * B, heads, kv, hd)
        sets.append(s)
        alone.append(run_attention(kc, *s))
    works = [kc.shared_attention_work(heads, kv, hd, B, R) for _ in sets]
    outs = [torch.zeros_like(a) for a in alone]
    at = torch.full((B,), S - R, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for s, w, o, stream in zip(sets, works, outs, streams):
            with torch.cuda.stream(stream):
                kc.k_attention_shared_rows(o, None, None, s[0], s[1], s[2], prefix, prefix, s[4], s[5], at, None, w, heads,
                                           kv, hd, S, B, R, 0)
    torch.cuda.synchronize()
    kc.status()
    for o, a, w in zip(outs, alone, works):
        assert torch.equal(o, a)
        kc.k_attention_free(w)


def test_mirror_refuses_what_does_not_fit(kc):
    """Tables and works that are too small for the call, types that are not the operator's: errors before any launch."""
    g = generator(3)
    x, out, index = normal(g, 4, 64), torch.zeros(4, 32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    table = kc.lora_table([normal(g, 8, 64)], [normal(g, 32, 8)], [1.0])
    with pytest.raises(kc.KernelError, match="2 adapters of a table of 1"):
        kc.k_lora_rows(out, 32, None, 0, x, 64, index, table, 2, kc.K_F32, 8, 64, 32, 4)
    for bad in (x.half(), x.cpu()):
        with pytest.raises(kc.KernelError, match="torch.float32 CUDA tensor on the current device"):
            kc.k_lora_rows(out, 32, None, 0, bad, 64, index, table, 1, kc.K_F32, 8, 64, 32, 4)
    with pytest.raises(kc.KernelError, match="torch.int32"):
        kc.k_lora_rows(out, 32, None, 0, x, 64, index.long(), table, 1, kc.K_F32, 8, 64, 32, 4)
    accepted, tokens = index[:1], torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    u, t, logits = torch.zeros(1, 2, device="cuda"), torch.ones(1, device="cuda"), normal(g, 2, 100)
    work = torch.zeros(kc.k_verify_bytes(100, 1, 1), dtype=torch.uint8, device="cuda")
    with pytest.raises(kc.KernelError, match="the work is too small"):
        kc.k_verify_draft(accepted, tokens, logits, 100, None, 0, tokens, None, u, t, 100, 1, 1, work[:-16])
    with pytest.raises(kc.KernelError, match="torch.float32 CUDA tensor"):
        kc.k_verify_draft(accepted, tokens, logits.half(), 100, None, 0, tokens, None, u, t, 100, 1, 1, work)


def test_nothing_to_do(kc):
    """A batch of none, rows of none: accepted, nothing queued."""
    before = kc.load().kc_launch_count()
    e = torch.empty(0, device="cuda")
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    kc.k_attention_shared_rows(e, None, None, e, e, e, 0, 0, e, e, i, i, kc.AttentionWork(), 8, 2, 64, 8, 0, 1, 0)
    kc.k_lora_rows(e, 8, e, 8, e, 8, i, None, 0, kc.K_F32, 8, 8, 8, 0)
    kc.k_verify_draft(i, i, e, 8, None, 0, i, i, e, e, 8, 0, 1, None)
    assert kc.load().kc_launch_count() == before
