"""KV caches in pages on the GPU against their numpy form (paged_ref.py): rows appended bit for bit, attention within the bar of f32 outputs, what is done
to pages exactly, and a run of all of it together with the picks of the next tokens."""
import numpy as np
import pytest

import paged_ref as R
import wick_amd as W
from conftest import assert_f32_parity
from wick_amd import lfm2
from wick_amd.lfm2 import KV_F16, KV_F32, KvPages, KvPlanes, Lfm2Ops, attention_paged_scratch_floats, kv_pages_moves_words

pytestmark = pytest.mark.gpu
NONE = R.NONE


@pytest.fixture()
def ops(ctx):
    return Lfm2Ops(ctx)


@pytest.fixture()
def dev(ctx):
    """Arrays to the device, freed behind the test."""
    bufs = []

    def put(a):
        bufs.append(ctx.to_device(a))
        return bufs[-1]

    yield put
    ctx.sync()
    for b in bufs:
        b.free()


def back(buf, like):
    return buf.download(like.dtype, like.size).reshape(like.shape)


def u32(*x):
    return np.array(x, np.int64).astype(np.uint32)


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


class OnDevice:
    """A Pool's arrays on the device."""

    def __init__(self, dev, pool):
        self.pool = pool
        self.table, self.lens, self.refs, self.planes = dev(pool.table), dev(u32(*pool.lens)), dev(pool.refs), dev(pool.planes)
        self.pages = KvPages(self.table, self.lens, self.refs, n_seqs=pool.S, max_pages=pool.max_pages, n_pages=pool.n_pages, page_rows=pool.R)
        self.plane_bytes = pool.planes[0].nbytes
        self.all = KvPlanes(self.planes, n_planes=len(pool.planes), plane_bytes=self.plane_bytes, n_kv_heads=pool.n_kv, head_dim=pool.hd, kv_dtype=pool.dtype)

    def plane(self, i):
        return self.planes.ptr + i * self.plane_bytes

    def check(self, planes=True):
        p = self.pool
        assert np.array_equal(back(self.table, p.table), p.table)
        assert np.array_equal(self.lens.download(np.uint32, p.S), u32(*p.lens))
        assert np.array_equal(back(self.refs, p.refs), p.refs)
        if planes:
            bits = {4: np.uint32, 2: np.uint16}[p.planes.itemsize]
            got = back(self.planes, p.planes)
            assert np.array_equal(got.view(bits), p.planes.view(bits)), np.argwhere(got.view(bits) != p.planes.view(bits))[:5]


def filled(seed, lens, page_rows, n_kv, hd, dtype, spare=3, shuffle=True, share=None):
    """A pool whose sequences hold rows of normal keys and values in pages of their own (share: {s: t}: s holds t's first pages too); all else is NaN."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page_rows) for n in lens]
    pool = R.Pool(len(lens), max(max(need), 1) + 1, sum(need) + spare, page_rows, n_kv, hd, dtype)
    ids = list(rng.permutation(pool.n_pages)) if shuffle else list(range(pool.n_pages))
    for s, n in enumerate(lens):
        pool.held[s], pool.lens[s] = [int(ids.pop(0)) for _ in range(need[s])], n
        for t in ([share[s]] if share and s in share else []):
            pool.held[s][:min(len(pool.held[t]), need[s]) - 1] = pool.held[t][:min(len(pool.held[t]), need[s]) - 1]
    for s, n in enumerate(lens):
        for plane in range(2):
            x = rng.standard_normal((n, n_kv, hd)).astype(R.TYPES[dtype])
            for i, page in enumerate(pool.held[s]):
                part = x[i * page_rows:(i + 1) * page_rows]
                pool.planes[plane, page, :, :len(part)] = part.transpose(1, 0, 2)
    return pool


def attend(ctx, ops, dev, d, q, extra=0, planes=(0, 1), scratch=None):
    """encode_attention_paged of q [S][heads][hd], with `extra` floats behind every row that have to stay."""
    p, (S, heads, hd) = d.pool, q.shape
    width = heads * hd + extra
    rows = np.full((S, width), 7.0, np.float32)
    rows[:, :heads * hd] = q.reshape(S, -1)
    out = np.full((S, width), 5.0, np.float32)
    d_out = dev(out)
    if scratch is None:
        scratch = dev(np.full(attention_paged_scratch_floats(S, heads, p.n_kv, hd), np.nan, np.float32))  # (contents need not be anything)
    ops.encode_attention_paged(d.pages, dev(rows), width, d.plane(planes[0]), d.plane(planes[1]), p.dtype, d_out, width, scratch, heads, p.n_kv, hd)
    got = back(d_out, out)
    assert np.all(got[:, heads * hd:] == 5.0)
    return got[:, :heads * hd].reshape(S, heads, hd)


# ---- append -----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("page_rows,n_kv,hd,extra", [(16, 8, 64, 0), (32, 1, 32, 4), (64, 3, 128, 64), (256, 2, 256, 0)])
def test_append_of_several_sequences(ops, dev, dtype, page_rows, n_kv, hd, extra):
    """Ragged tokens: none of a sequence, one, many; a sequence whose tokens are dropped; rows past its pages and past the table."""
    lens = [page_rows + 5, 2 * page_rows, 40, 3, page_rows - 1]
    pool = filled(1, lens, page_rows, n_kv, hd, dtype)
    d = OnDevice(dev, pool)
    counts, start = [3, 0, 30, 7, 2 * page_rows + 9], [page_rows - 2, 0, 10, NONE, page_rows - 1]
    first = np.concatenate([[0], np.cumsum(counts)])
    n = int(first[-1]) + 2  # (two tokens that are nobody's)
    k, v = normal(2, n, n_kv * hd + extra), normal(3, n, n_kv * hd + extra) * 100
    k[0, 0], v[1, 1], k[2, 2], k[3, 3], v[3, 0] = np.inf, np.nan, 65520.0, 1e-8, -0.0
    ops.encode_kv_paged_append(d.pages, dev(k), dev(v), n_kv * hd + extra, d.plane(0), d.plane(1), dtype, dev(u32(*start)), n, n_kv, hd, first=dev(u32(*first)))
    for s in range(5):
        for i in range(counts[s] if start[s] != NONE else 0):
            j = first[s] + i
            pool.put(s, start[s] + i, k[j, :n_kv * hd].reshape(n_kv, hd), v[j, :n_kv * hd].reshape(n_kv, hd))
    got = back(d.planes, pool.planes)
    assert np.array_equal(got, pool.planes, equal_nan=True) and np.array_equal(np.signbit(got), np.signbit(pool.planes))


@pytest.mark.parametrize("seqs", [1, 70, 4096])
def test_append_of_one_token_each(ops, dev, seqs):
    lens = [1 + s % 40 for s in range(seqs)]
    pool = filled(4, lens, 16, 1, 32, KV_F16)
    d = OnDevice(dev, pool)
    k, v = normal(5, seqs, 32), normal(6, seqs, 32)
    ops.encode_kv_paged_append(d.pages, dev(k), dev(v), 32, d.plane(0), d.plane(1), KV_F16, dev(u32(*(n - 1 for n in lens))), seqs, 1, 32)
    for s in range(seqs):
        pool.put(s, lens[s] - 1, k[s].reshape(1, 32), v[s].reshape(1, 32))
    d.check()


def test_appended_rows_without_a_page_are_dropped(ops, dev):
    """Entries that name no page, and pages that are not the pool's."""
    pool = filled(7, [40, 40, 40], 16, 2, 64, KV_F32)
    table = pool.table
    d = OnDevice(dev, pool)
    table[0, 2], table[1, 2], table[2, 2] = NONE, pool.n_pages, 0x7fffffff
    d.table.upload(table)
    x = normal(8, 3, 128)
    ops.encode_kv_paged_append(d.pages, dev(x), dev(x), 128, d.plane(0), d.plane(1), KV_F32, dev(u32(39, 39, 39)), 3, 2, 64)
    for row in (1 << 20, NONE - 1):
        ops.encode_kv_paged_append(d.pages, dev(x), dev(x), 128, d.plane(0), d.plane(1), KV_F32, dev(u32(row, row, row)), 3, 2, 64)
    assert np.array_equal(back(d.planes, pool.planes), pool.planes, equal_nan=True)


# ---- tokens normed, rotated and appended ------------------------------------------------------------

@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("heads,n_kv,hd,page_rows,pad,one_each", [
    (16, 8, 64, 16, 0, False), (4, 2, 64, 64, 3, True), (40, 8, 64, 32, 0, True), (3, 3, 128, 32, 5, False), (6, 2, 256, 16, 0, True), (17, 1, 32, 256, 1, False)])
def test_tokens_of_several_sequences_normed_and_rotated(ctx, ops, dev, dtype, heads, n_kv, hd, page_rows, pad, one_each):
    """One launch for tokens at rows of their own as wick_rocm_qk_norm_rope and wick_rocm_kv_paged_append token by token, bit for bit; few tokens and many."""
    eps, ts, kv_dim = 1e-5, lfm2.rope_theta_scale(hd, 1_000_000.0), n_kv * hd
    counts = [1] * 9 if one_each else [3, 0, 300, 1, 40]
    lens = [500, 3, 0, 15, 16, 17, 31, 700, 1][:len(counts)]
    n, S = sum(counts), len(counts)
    pool = filled(50, [a + b for a, b in zip(lens, counts)], page_rows, n_kv, hd, dtype)
    d, d2 = OnDevice(dev, pool), OnDevice(dev, pool)
    start = u32(*lens)
    start[1] = NONE  # sequence 1's are dropped
    table = pool.table
    table[4, lens[4] // page_rows] = NONE  # there is no page for the first of sequence 4's
    for x in (d, d2):
        x.table.upload(table)
    width = heads * hd + 2 * kv_dim + pad  # one [q | k | v] row a token
    rows = normal(51, n + 2, width)  # two more tokens than there are: of no sequence
    first = u32(0, *np.cumsum(counts))
    d_rows, d_rows2, qn, kn, none = dev(rows), dev(rows), dev(1 + 0.2 * normal(52, hd)), dev(1 + 0.2 * normal(53, hd)), dev(np.zeros(kv_dim, np.float32))

    def parts(r, j=0):
        p = r.ptr + 4 * j * width
        return p, p + 4 * heads * hd, p + 4 * (heads * hd + kv_dim)

    q, k, v = parts(d_rows)
    ops.encode_qk_norm_rope_paged(d.pages, q, width, k, v, width, qn, kn, d.plane(0), d.plane(1), dtype, dev(start), n if one_each else n + 2, heads, n_kv, hd, eps, ts,
                                  first=None if one_each else dev(first))
    got = back(d_rows, rows)
    for s in range(S):
        for i in range(counts[s] if start[s] != NONE else 0):
            j = int(first[s]) + i
            # (a position at or behind its cache's rows is not stored)
            q, k, v = parts(d_rows2, j)
            ops.encode_qk_norm_rope(q, k, v, qn, kn, none, none, 0, 0, hd, heads, n_kv, eps, ts, d_pos=dev(u32(lens[s] + i)))
            one = u32(*[NONE] * S)
            one[s] = lens[s] + i
            kv = back(d_rows2, rows)[j, heads * hd:heads * hd + 2 * kv_dim]
            ops.encode_kv_paged_append(d2.pages, dev(kv[:kv_dim]), dev(kv[kv_dim:]), kv_dim, d2.plane(0), d2.plane(1), dtype, dev(one), 1, n_kv, hd,
                                       first=dev(u32(*[0] * (s + 1), *[1] * (S - s))))
    want = back(d_rows2, rows)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32)) and not np.array_equal(got, rows)
    assert np.array_equal(got[n:], rows[n:]) and np.array_equal(got[first[1]:first[2]], rows[first[1]:first[2]])
    bits = {4: np.uint32, 2: np.uint16}[pool.planes.itemsize]
    a, b = back(d.planes, pool.planes).view(bits), back(d2.planes, pool.planes).view(bits)
    assert np.array_equal(a, b) and not np.array_equal(a, pool.planes.view(bits))


# ---- attention -----------------------------------------------------------------------------------

ATTENTION = [  # head_dim, heads, KV heads, page_rows, lengths
    (64, 16, 8, 16, [1]), (64, 16, 8, 16, [701]), (64, 16, 8, 64, [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 0]), (64, 32, 8, 32, [5000, 3, 0, 77, 1200]),
    (64, 8, 8, 128, [300, 299]), (64, 24, 3, 256, [1000, 2]), (64, 16, 1, 16, [64, 700]), (64, 17, 1, 16, [64, 700]), (64, 64, 2, 32, [333] * 3), (64, 50, 2, 16, [1, 4000]),
    (32, 4, 2, 16, [77, 100, 2]), (32, 40, 1, 64, [5000]), (128, 8, 2, 16, [129, 640]), (128, 32, 8, 64, [3001]), (128, 5, 5, 32, [1, 33, 65]), (256, 4, 1, 16, [33]),
    (256, 6, 2, 64, [2500, 0, 12]), (256, 32, 1, 128, [900]), (32, 1, 1, 16, [20000]), (64, 16, 8, 16, list(range(0, 300, 3))),
]


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("hd,heads,n_kv,page_rows,lens", ATTENTION, ids=[f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}" for c in ATTENTION])
def test_attention(ctx, ops, dev, hd, heads, n_kv, page_rows, lens, dtype):
    """Rows that no sequence has hold NaN, and so does the scratch."""
    pool = filled(len(lens) + hd, lens, page_rows, n_kv, hd, dtype)
    q = normal(11, len(lens), heads, hd) * 1.5
    got = attend(ctx, ops, dev, OnDevice(dev, pool), q, extra=4 * (len(lens) % 3))
    want = pool.attention(q)
    assert_f32_parity(got, want)
    assert np.all(got[np.array(lens) == 0] == 0)
    for s, n in enumerate(lens):  # every sequence by itself: a long one does not hide a short one
        if n:
            assert_f32_parity(got[s], want[s], f"sequence {s}")


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_attention_of_many_sequences(ctx, ops, dev, dtype):
    lens = [int(n) for n in np.random.default_rng(3).integers(0, 40, 4096)]
    lens[4095], lens[0] = 200, 0
    pool = filled(12, lens, 16, 1, 32, dtype)
    q = normal(13, 4096, 2, 32)
    assert_f32_parity(attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q))


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("hd,heads,n_kv,page_rows,lens", ATTENTION, ids=[f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}" for c in ATTENTION])
def test_attention_under_a_wide_table(ctx, ops, dev, hd, heads, n_kv, page_rows, lens, dtype):
    """Room for many more rows than there are: what is taken in one launch above is split over shares and joined."""
    pool = filled(len(lens) + hd, lens, page_rows, n_kv, hd, dtype)
    pool.max_pages += 2048 // page_rows
    q = normal(11, len(lens), heads, hd) * 1.5
    got = attend(ctx, ops, dev, OnDevice(dev, pool), q, extra=4)
    want = pool.attention(q)
    for s, n in enumerate(lens):
        assert_f32_parity(got[s], want[s], f"sequence {s}") if n else np.testing.assert_array_equal(got[s], 0)


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("longest,spread", [(40, 1), (2, 1), (40, 500)])
def test_attention_of_many_sequences_under_a_wide_table(ctx, ops, dev, dtype, longest, spread):
    """4096 sequences, of which all, or one in 500, have rows: the others lie between those that a share has."""
    lens = [int(n) if s % spread == 0 else 0 for s, n in enumerate(np.random.default_rng(36).integers(0, longest, 4096))]
    lens[4095], lens[2001] = 200, 2500
    pool = filled(37, lens, 16, 2, 32, dtype)
    pool.max_pages = 300
    q = normal(38, 4096, 4, 32)
    got, want = attend(ctx, ops, dev, OnDevice(dev, pool), q, extra=4), pool.attention(q)
    assert_f32_parity(got, want)
    assert np.all(got[np.array(lens) == 0] == 0)
    for s in (2001, 4095):
        assert_f32_parity(got[s], want[s])


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("seqs,hd,heads,n_kv", [(600, 32, 1, 1), (130, 64, 8, 4), (40, 64, 40, 8), (300, 128, 17, 1), (70, 256, 4, 4)])
def test_more_heads_than_shares(ctx, ops, dev, dtype, seqs, hd, heads, n_kv):
    """Sequences of all lengths and of none, also at both ends; heads that end where a share does and heads over several shares."""
    lens = [int(n) for n in np.random.default_rng(seqs).integers(0, 400, seqs)]
    for s in (0, 7, 8, 70, seqs - 1):
        lens[s % seqs] = 0
    lens[1], lens[seqs // 2] = 128, 3000
    pool = filled(34, lens, 64, n_kv, hd, dtype)
    q = normal(35, seqs, heads, hd)
    got, want = attend(ctx, ops, dev, OnDevice(dev, pool), q, extra=8), pool.attention(q)
    for s, n in enumerate(lens):
        assert_f32_parity(got[s], want[s], f"sequence {s}") if n else np.testing.assert_array_equal(got[s], 0)


def test_attention_over_shared_pages(ctx, ops, dev):
    pool = filled(14, [900, 901, 400, 33], 32, 2, 64, KV_F16, share={1: 0, 2: 0, 3: 1})
    q = normal(15, 4, 8, 64)
    assert pool.refs.max() >= 3
    assert_f32_parity(attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q))


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_rows_without_a_page_are_not_there(ctx, ops, dev, dtype):
    """In the middle, at both ends, all of them (zeros); page 0, which is read in their place, holds NaN."""
    pool = filled(16, [200, 100, 64, 700], 16, 2, 64, dtype, shuffle=False)
    pool.held = [[p + 1 for p in h] for h in pool.held]
    pool.planes = np.concatenate([np.full_like(pool.planes[:, :1], np.nan), pool.planes[:, :-1]], 1)
    table, seen = pool.table, {s: np.ones(n, bool) for s, n in enumerate(pool.lens)}
    for s, pages in enumerate(([3, 4, 12], [0, 6], range(4), [1, 40])):
        for i, p in enumerate(pages):
            table[s, p] = (NONE, pool.n_pages, 0x80000000)[i % 3]
            seen[s][16 * p:16 * p + 16] = False
    d = OnDevice(dev, pool)
    d.table.upload(table)
    q = normal(17, 4, 4, 64)
    got = attend(ctx, ops, dev, d, q)
    want = pool.attention(q, seen=seen)
    assert np.all(got[2] == 0) and np.all(want[2] == 0)
    for s in (0, 1, 3):
        assert_f32_parity(got[s], want[s])


def test_lengths_past_the_table_are_its_rows(ctx, ops, dev):
    pool = filled(18, [64, 64], 16, 1, 64, KV_F16, spare=0)
    pool.max_pages = 4
    d = OnDevice(dev, pool)
    d.lens.upload(u32(64, 4000000000))
    q = normal(19, 2, 4, 64)
    assert_f32_parity(attend(ctx, ops, dev, d, q), pool.attention(q))


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_a_row_that_is_not_finite_stays_with_those_that_read_it(ctx, ops, dev, dtype):
    pool = filled(20, [300, 300, 170, 170], 32, 2, 64, dtype)
    pool.planes[0, pool.held[0][3], 1, 5, 7] = np.nan  # a key of sequence 0, KV head 1
    pool.planes[1, pool.held[1][0], 0, 2, 9] = np.inf  # a value of sequence 1, KV head 0
    q = normal(21, 4, 4, 64)
    got = attend(ctx, ops, dev, OnDevice(dev, pool), q)
    with np.errstate(invalid="ignore"):
        want = pool.attention(q)
    assert np.isnan(got[0, 2:]).all() and not np.isfinite(got[1, :2, 9]).any()
    clean = np.isfinite(want)
    assert np.isfinite(got[0, :2]).all() and np.isfinite(got[1, 2:]).all() and np.isfinite(got[2:]).all()
    assert clean[2:].all()
    for s, h in ((0, 0), (0, 1), (1, 2), (1, 3), (2, 0), (3, 3)):
        assert_f32_parity(got[s, h], want[s, h])


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-30, 1e-3, 1.0, 5.0])
def test_queries_of_every_size(ctx, ops, dev, dtype, scale):
    pool = filled(22, [150, 20], 16, 2, 64, dtype)
    q = normal(23, 2, 6, 64) * np.float32(scale)
    q[:, 0, 1:] *= np.float32(1e-4)  # one element far above the others
    q[0, 1] = 0
    assert_f32_parity(attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q))


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_large_keys_under_small_queries(ctx, ops, dev, dtype):
    """Channels of the keys that are 1000 times as large as the others, the queries' as small."""
    pool = filled(24, [400], 16, 1, 128, dtype)
    q = normal(25, 1, 8, 128)
    pool.planes[0, ..., :4] *= 1000
    q[..., :4] /= 1000
    assert_f32_parity(attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q))


@pytest.mark.parametrize("at", [0, 100, 699])
@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_one_row_that_draws_all(ctx, ops, dev, dtype, at):
    """A score far above the others, first, in the middle and last: the state is scaled down, or what follows is next to nothing."""
    pool = filled(26, [700, 700], 16, 2, 64, dtype)
    q = normal(27, 2, 4, 64)
    for c in range(2):
        pool.planes[0, pool.held[0][at // 16], c, at % 16] = 20 * q[0, 2 * c]
    assert_f32_parity(attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q))


def test_pages_past_two_and_four_gib(ctx, ops, dev):
    """A pool of 9.7 GB a plane whose rows in use lie at its far end."""
    n_pages, page_rows, n_kv, hd = 37000, 64, 8, 256
    small = filled(28, [200, 64], page_rows, n_kv, hd, KV_F16, spare=0)
    far = n_pages - small.n_pages
    nbytes = n_pages * n_kv * page_rows * hd * 2
    planes = [ctx.alloc(nbytes) for _ in range(2)]
    try:
        for plane, x in zip(planes, small.planes):
            plane.upload(x, offset_bytes=far * n_kv * page_rows * hd * 2)
        table = np.where(small.table == NONE, NONE, small.table + np.uint32(far)).astype(np.uint32)
        pages = KvPages(dev(table), dev(u32(*small.lens)), dev(np.zeros(n_pages, np.uint32)), n_seqs=2, max_pages=small.max_pages, n_pages=n_pages, page_rows=page_rows)
        k, v = normal(29, 2, n_kv * hd), normal(30, 2, n_kv * hd)
        ops.encode_kv_paged_append(pages, dev(k), dev(v), n_kv * hd, *planes, KV_F16, dev(u32(199, 63)), 2, n_kv, hd)
        for s in range(2):
            small.put(s, small.lens[s] - 1, k[s].reshape(n_kv, hd), v[s].reshape(n_kv, hd))
        q = normal(31, 2, 16, hd)
        d_out = dev(np.zeros((2, 16 * hd), np.float32))
        scratch = dev(np.zeros(attention_paged_scratch_floats(2, 16, n_kv, hd), np.float32))
        ops.encode_attention_paged(pages, dev(q), 16 * hd, *planes, KV_F16, d_out, 16 * hd, scratch, 16, n_kv, hd)
        assert_f32_parity(back(d_out, q), small.attention(q))
        # the last page to the first, in both planes (they are not apart by one stride: one by one)
        moves = np.zeros(8, np.uint32)
        moves[:7] = [1, 0, 0, 0, n_pages - 1, 1, page_rows]
        for plane, x in zip(planes, small.planes):
            ops.kv_pages_copy(pages, KvPlanes(plane, n_planes=1, plane_bytes=0, n_kv_heads=n_kv, head_dim=hd, kv_dtype=KV_F16), dev(moves), 1)
            size = n_kv * page_rows * hd
            assert np.array_equal(plane.download(np.float16, size, offset_bytes=2 * size), x[-1].ravel(), equal_nan=True)
    finally:
        ctx.sync()
        for p in planes:
            p.free()


def test_attention_gives_the_same_bits_in_every_run(ctx, ops, dev):
    pool = filled(32, [3000, 17, 0, 800], 16, 4, 64, KV_F16)
    q = normal(33, 4, 16, 64)
    d = OnDevice(dev, pool)
    runs = [attend(ctx, ops, dev, d, q) for _ in range(3)]
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


# ---- pages ------------------------------------------------------------------------------------------

def moves_of(d_moves):
    head = d_moves.download(np.uint32, 4)
    return [tuple(m[:3]) for m in d_moves.download(np.uint32, 4 * int(head[0]), offset_bytes=16).reshape(-1, 4).tolist()], int(head[1])


@pytest.mark.parametrize("dtype,n_kv,hd,page_rows", [(KV_F16, 2, 64, 16), (KV_F32, 1, 32, 16), (KV_F16, 3, 32, 64), (KV_F32, 1, 128, 32), (KV_F16, 1, 256, 256)])
@pytest.mark.parametrize("seed", range(4))
def test_a_life_of_pages(ctx, ops, dev, dtype, n_kv, hd, page_rows, seed):
    """Sequences that fork, grow, are cut, leave and are moved together, at random: table, lens, refs and every byte of the planes as the lists have them."""
    rng = np.random.default_rng(100 * seed + hd)
    pool = R.Pool(int(rng.integers(1, 9)), 9, 24, page_rows, n_kv, hd, dtype, n_planes=3)
    pool.planes[:] = rng.standard_normal(pool.planes.shape)
    d = OnDevice(dev, pool)
    start, moves = dev(np.zeros(pool.S, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
    seen = set()
    for step in range(40):
        what = rng.choice(["reserve", "reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            counts = [int(c) for c in rng.integers(0, 1 + int(rng.choice([1, 5, 2 * page_rows])), pool.S)]
            want, copied, wanting = pool.reserve(counts)
            pool.copy(copied)
            ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves, d.all)
            got, said = moves_of(moves)
            assert said == wanting and sorted(got) == sorted(copied), (step, counts)
            assert np.array_equal(start.download(np.uint32, pool.S), u32(*want))
            seen.add("refused" if wanting else "copied" if copied else "reserved")
        elif what == "fork":
            parents = [int(p) for p in rng.integers(0, pool.S + 1, pool.S)]
            parents = [s if rng.random() < 0.5 else NONE if p == pool.S else p for s, p in enumerate(parents)]
            pool.fork(parents)
            ops.kv_pages_fork(d.pages, dev(u32(*parents)))
        elif what == "free":
            rows = [int(r) for r in rng.choice([0, 1, page_rows - 1, page_rows, page_rows + 1, 3 * page_rows, 100000, NONE], pool.S)]
            pool.free(rows)
            ops.kv_pages_free(d.pages, dev(u32(*rows)))
        else:
            moved, used = pool.compact()
            pool.copy(moved)
            ops.kv_pages_compact(d.pages, moves, d.all)
            assert moves_of(moves) == (moved, used)
        d.check()
    assert "reserved" in seen


def test_the_first_of_those_that_share_a_page_alone_keeps_it(ops, dev):
    """Four hold a partial page: all write, the first keeps it; three write, all three copy; one is alone, nothing is copied."""
    for counts, copied in (([1, 2, 3, 4], [1, 2, 3]), ([0, 1, 1, 1], [1, 2, 3]), ([0, 0, 5, 0], [2])):
        pool = R.Pool(4, 8, 40, 16, 2, 64, KV_F16)
        pool.planes[:] = normal(40, *pool.planes.shape)
        pool.reserve([20, 0, 0, 0])
        pool.fork([0, 0, 0, 0])
        d = OnDevice(dev, pool)
        start, moves = dev(np.zeros(4, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
        _, want, _ = pool.reserve(counts)
        pool.copy(want)
        ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves, d.all)
        assert len(want) == len(copied) and all(pool.held[s][1] != 1 for s in copied)
        d.check()
    pool.free([0, 0, 1000, 0])
    d = OnDevice(dev, pool)
    _, want, _ = pool.reserve([0, 0, 1, 0])
    ops.kv_pages_reserve(d.pages, dev(u32(0, 0, 1, 0)), start, moves, d.all)
    assert want == []
    d.check()


@pytest.mark.parametrize("max_pages,n_pages", [(4, 9), (8, 7)])
def test_a_reservation_that_does_not_fit_changes_nothing(ops, dev, max_pages, n_pages):
    """Where the tables are too short, and where the pool has not enough; what does fit goes through before and behind it."""
    pool = R.Pool(3, max_pages, n_pages, 16, 1, 32, KV_F32)
    pool.planes[:] = normal(41, *pool.planes.shape)
    pool.reserve([40, 0, 0])
    pool.fork([0, 0, 0])
    d = OnDevice(dev, pool)
    start, moves = dev(np.zeros(3, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
    outcomes = []
    for counts in ([20, 20, 20], [24, 24, 24], [8, 8, 24], [64, 0, 0], [25, 0, 0], [NONE, 1, 1], [1, 0, 1]):
        said = pool.reserve(list(counts))
        pool.copy(said[1])
        ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves, d.all)
        assert moves_of(moves)[1] == said[2]
        assert np.array_equal(start.download(np.uint32, 3), u32(*said[0]))
        d.check()
        outcomes.append("table" if said[2] == NONE else "pool" if said[2] else "fits")
    assert {"fits", "table" if max_pages == 4 else "pool"} <= set(outcomes), outcomes


def test_many_pages_and_sequences(ops, dev):
    """4096 sequences in a pool of 70000 pages, with holes all over; bookkeeping alone, then the moves by a call of their own."""
    rng = np.random.default_rng(5)
    pool = R.Pool(4096, 40, 70000, 16, 1, 32, KV_F16, n_planes=1)
    pool.planes = np.arange(70000, dtype=np.uint16).repeat(16 * 32).view(np.float16).reshape(1, 70000, 1, 16, 32)
    d = OnDevice(dev, pool)
    start, moves = dev(np.zeros(4096, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
    for round_ in range(3):
        counts = [int(c) for c in rng.integers(0, 200, 4096)]
        want, copied, wanting = pool.reserve(counts)
        assert wanting == 0
        ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves)
        got, said = moves_of(moves)
        assert said == 0 and sorted(got) == sorted(copied)
        assert np.array_equal(start.download(np.uint32, 4096), u32(*want))
        ops.kv_pages_copy(d.pages, d.all, moves, 4096)
        pool.copy(copied)
        parents = [int(p) if rng.random() < 0.3 else s for s, p in enumerate(rng.integers(0, 5000, 4096))]
        pool.fork(parents)
        ops.kv_pages_fork(d.pages, dev(u32(*parents)))
        d.check(planes=False)
        moved, used = pool.compact()
        ops.kv_pages_compact(d.pages, moves)
        assert moves_of(moves) == (moved, used)
        ops.kv_pages_copy(d.pages, d.all, moves, len(moved))
        pool.copy(moved)
        d.check()


def test_copies_of_a_list(ops, dev):
    """No more than max_moves; rows in part, more rows than a page has, pages that are none."""
    pool = R.Pool(1, 4, 12, 32, 2, 64, KV_F16, n_planes=4)
    pool.planes[:] = normal(42, *pool.planes.shape)
    d = OnDevice(dev, pool)
    listed = [(0, 5, 32), (1, 6, 1), (2, 7, 0), (3, 8, 100), (12, 9, 32), (4, NONE, 32), (4, 10, 31), (4, 11, 32)]
    words = np.zeros(4 + 4 * len(listed), np.uint32)
    words[0] = len(listed)
    for i, m in enumerate(listed):
        words[4 + 4 * i:7 + 4 * i] = m
    ops.kv_pages_copy(d.pages, d.all, dev(words), 7)
    pool.copy([(a, b, min(r, 32)) for a, b, r in listed[:7] if a < 12 and b < 12])
    d.check()
    ops.kv_pages_copy(d.pages, d.all, dev(words), 0)
    d.check()


def test_page_calls_on_an_empty_pool(ops, dev):
    pool = R.Pool(5, 3, 7, 16, 1, 32, KV_F16)
    d = OnDevice(dev, pool)
    start, moves = dev(np.zeros(5, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
    ops.kv_pages_compact(d.pages, moves, d.all)
    assert moves_of(moves) == ([], 0)
    ops.kv_pages_fork(d.pages, dev(u32(1, 2, 3, 4, 0)))
    ops.kv_pages_free(d.pages, dev(u32(0, 0, 0, 0, 0)))
    ops.kv_pages_reserve(d.pages, dev(u32(0, 0, 0, 0, 0)), start, moves, d.all)
    assert moves_of(moves) == ([], 0) and np.all(start.download(np.uint32, 5) == NONE)
    d.check()


# ---- together -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_continuations_of_a_prompt(ctx, ops, dev, dtype):
    """A prompt's rows (as the contiguous caches have them) appended, continued several times -- forked, one of the branches dropped, the pool moved together --
    with attention of every step as over contiguous caches of the same rows, by wick_rocm_attention_decode, and picks from the outputs."""
    heads, n_kv, hd, page_rows, branches, max_seq = 8, 2, 64, 16, 5, 128
    pool = R.Pool(branches, 8, 40, page_rows, n_kv, hd, dtype)
    d = OnDevice(dev, pool)
    start, moves = dev(np.zeros(branches, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
    scratch = dev(np.zeros(attention_paged_scratch_floats(branches, heads, n_kv, hd), np.float32))
    scores = dev(np.zeros(lfm2.attention_scratch_floats(max_seq, heads, hd), np.float32))
    held = [np.zeros((2, 0, n_kv * hd), np.float32) for _ in range(branches)]  # what every branch has appended

    def append(counts, seed):
        n = sum(counts)
        k, v = normal(seed, n, n_kv * hd), normal(seed + 1, n, n_kv * hd)
        first = u32(0, *np.cumsum(counts))
        ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves, d.all)
        ops.encode_kv_paged_append(d.pages, dev(k), dev(v), n_kv * hd, d.plane(0), d.plane(1), dtype, start, n, n_kv, hd, first=dev(first))
        for s in range(branches):
            held[s] = np.concatenate([held[s], np.stack([k, v])[:, first[s]:first[s + 1]]], 1)

    def check(seed):
        q = normal(seed, branches, heads, hd)
        got = attend(ctx, ops, dev, d, q, scratch=scratch)
        for s in range(branches):
            n = held[s].shape[1]
            rows = np.zeros((2, max_seq, n_kv * hd), np.float32)
            rows[:, :n] = held[s].astype(R.TYPES[dtype])  # (f16 pages: rounded once)
            want = np.zeros(heads * hd, np.float32)
            d_want = dev(want)
            if n:
                ops.encode_attention(dev(q[s]), dev(rows[0]), dev(rows[1]), d_want, scores, n, max_seq, heads, n_kv, hd)
                want = back(d_want, want)
            assert_f32_parity(got[s].ravel(), want, f"branch {s} of {n} rows")
        logits = got.reshape(branches, -1)
        token, prob = dev(np.zeros(branches, np.uint32)), dev(np.zeros(branches, np.float32))
        u = np.random.default_rng(seed).random(branches).astype(np.float32)
        params = [(0.5, 20, 0.9, 0.0)] * branches
        ops.sample(dev(logits), logits.shape[1], branches, logits.shape[1], dev(lfm2.sample_params(params).view(np.uint32)), dev(u), token, prob,
                   dev(np.zeros(lfm2.sample_scratch_bytes(branches, logits.shape[1]), np.uint8)))
        for s in range(branches):
            want = R.sample(logits[s], *params[s], u[s])
            assert token.download(np.uint32, branches)[s] == want[0] or want[2] < 1e-6

    append([37, 0, 0, 0, 0], 50)
    check(51)
    ops.kv_pages_fork(d.pages, dev(u32(0, 0, 0, 0, NONE)))
    held[1] = held[2] = held[3] = held[0]
    for step in range(4):
        append([1, 1, 1, 1, 0], 60 + 10 * step)
        check(61 + 10 * step)
    ops.kv_pages_free(d.pages, dev(u32(1000, 0, 38, 1000, 0)))
    held[1], held[2] = held[1][:, :0], held[2][:, :38]
    ops.kv_pages_compact(d.pages, moves, d.all)
    check(120)
    append([3, 20, 1, 17, 5], 130)
    check(131)
    ops.kv_pages_fork(d.pages, dev(u32(3, 1, 0, 4, 2)))
    held = [held[i] for i in (3, 1, 0, 4, 2)]
    append([1] * 5, 140)
    check(141)
    used = len({p for row in back(d.table, pool.table).tolist() for p in row if p != NONE})
    assert (back(d.refs, pool.refs) > 0).sum() == used


def test_steps_of_sessions_as_each_by_itself(ctx, ops, dev):
    """The attention block of several steps of five sessions at once -- rows reserved, tokens normed, rotated and appended, attention -- against
    wick_rocm_attention_block of each over a cache of its own; one session sits out a step, one ends."""
    heads, n_kv, hd, max_seq, eps = 16, 4, 64, 256, 1e-5
    S, kv_dim, width, ts = 5, n_kv * hd, heads * hd + 2 * n_kv * hd, lfm2.rope_theta_scale(hd, 1_000_000.0)
    pool = R.Pool(S, 8, 30, 16, n_kv, hd, KV_F32)
    d = OnDevice(dev, pool)
    start, moves = dev(np.zeros(S, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
    scratch, sc = dev(np.zeros(attention_paged_scratch_floats(S, heads, n_kv, hd), np.float32)), dev(np.zeros(lfm2.attention_block_scratch_bytes(max_seq, heads, hd), np.uint8))
    qn, kn = dev(1 + 0.2 * normal(60, hd)), dev(1 + 0.2 * normal(61, hd))
    caches, rows_of = [[dev(np.zeros(max_seq * kv_dim, np.float32)) for _ in range(2)] for _ in range(S)], [0] * S
    out, one = dev(np.zeros((S, heads * hd), np.float32)), dev(np.zeros(heads * hd, np.float32))
    for step in range(40):
        counts = [int(not (s == step % 7 and step % 2)) for s in range(S)]
        if step == 25:
            ops.kv_pages_free(d.pages, dev(u32(NONE, NONE, 0, NONE, NONE)))
            ops.kv_pages_compact(d.pages, moves, d.all)
            rows_of[2] = 0
        x = normal(100 + step, S, width)
        ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves, d.all)
        d_x = dev(x)
        q, k, v = d_x.ptr, d_x.ptr + 4 * heads * hd, d_x.ptr + 4 * (heads * hd + kv_dim)
        ops.encode_qk_norm_rope_paged(d.pages, q, width, k, v, width, qn, kn, d.plane(0), d.plane(1), KV_F32, start, S, heads, n_kv, hd, eps, ts)
        ops.encode_attention_paged(d.pages, q, width, d.plane(0), d.plane(1), KV_F32, out, heads * hd, scratch, heads, n_kv, hd)
        got = out.download(np.float32, S * heads * hd).reshape(S, -1)
        for s in range(S):
            if not counts[s]:
                continue
            o = [dev(np.ascontiguousarray(p)) for p in np.split(x[s], [heads * hd, heads * hd + kv_dim])]
            ops.encode_attention_block(o[0], o[1], o[2], qn, kn, caches[s][0], caches[s][1], one, sc, rows_of[s], max_seq, hd, heads, n_kv, eps, ts)
            rows_of[s] += 1
            assert_f32_parity(got[s], one.download(np.float32, heads * hd), f"step {step}, session {s}")


def test_a_captured_step_replayed(ctx, ops, dev):
    """reserve, append, attention and the pick of every sequence's next token as one graph, replayed with eager work between, against the same calls one by one."""
    S, heads, n_kv, hd = 3, 8, 2, 64
    width = heads * hd
    params, k, v, q = lfm2.sample_params([(0.7, 0, 0.95, 0.0)] * S).view(np.uint32), normal(70, S, n_kv * hd), normal(71, S, n_kv * hd), normal(72, S, width)
    u = np.array([0.1, 0.5, 0.9], np.float32)
    ones = u32(1, 1, 1)
    scratch, picks = dev(np.zeros(attention_paged_scratch_floats(S, heads, n_kv, hd), np.float32)), dev(np.zeros(lfm2.sample_scratch_bytes(S, width), np.uint8))
    d_params, d_k, d_v, d_q, d_u, d_ones = (dev(x) for x in (params, k, v, q, u, ones))

    def make():
        pool = R.Pool(S, 9, 30, 16, n_kv, hd, KV_F16)
        pool.planes[:] = normal(73, *pool.planes.shape)
        pool.reserve([30, 0, 0])
        pool.fork([0, 0, 0])
        d = OnDevice(dev, pool)
        return d, dev(np.zeros(S, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32)), dev(np.zeros((S, width), np.float32)), dev(np.zeros(S, np.uint32)), dev(
            np.zeros(S, np.float32))

    def step(d, start, moves, out, token, prob):
        ops.kv_pages_reserve(d.pages, d_ones, start, moves, d.all)
        ops.encode_kv_paged_append(d.pages, d_k, d_v, n_kv * hd, d.plane(0), d.plane(1), KV_F16, start, S, n_kv, hd)
        ops.encode_attention_paged(d.pages, d_q, width, d.plane(0), d.plane(1), KV_F16, out, width, scratch, heads, n_kv, hd)
        ops.sample(out, width, S, width, d_params, d_u, token, prob, picks)

    def seen(d, start, moves, out, token, prob):
        return [b.download(np.uint8, b.nbytes) for b in (d.table, d.lens, d.refs, d.planes, start, out, token, prob)]

    eager, replayed = make(), make()
    ctx.graph_begin()
    step(*replayed)
    g = ctx.graph_end()
    for _ in range(20):  # over the end of a page
        step(*eager)
        want = seen(*eager)
        ctx.graph_launch(g)
        ctx.sync()
        assert all(np.array_equal(a, b) for a, b in zip(want, seen(*replayed)))
    ctx.graph_destroy(g)


def test_two_contexts_at_once(ctx, dev):
    """Two sessions' steps in flight together, each with a pool and scratch of its own."""
    with W.RocmContext(0) as other:
        ops, sides = [Lfm2Ops(ctx), Lfm2Ops(other)], []
        for i in range(2):
            pool = filled(80 + i, [900, 30, 2000], 16, 4, 64, KV_F16)
            q = normal(82 + i, 3, 16, 64)
            d = OnDevice(dev, pool)
            sides.append((pool, d, q, dev(q), dev(np.zeros_like(q)), dev(np.zeros(attention_paged_scratch_floats(3, 16, 4, 64), np.float32))))
        for _ in range(10):
            for op, (_, d, _, d_q, d_out, scratch) in zip(ops, sides):
                op.encode_attention_paged(d.pages, d_q, 1024, d.plane(0), d.plane(1), KV_F16, d_out, 1024, scratch, 16, 4, 64)
        ctx.sync(), other.sync()
        for pool, _, q, _, d_out, _ in sides:
            assert_f32_parity(back(d_out, q), pool.attention(q))


@pytest.mark.parametrize("hd,heads,n_kv,page_rows", [(64, 8, 2, 16), (32, 3, 3, 32), (128, 8, 1, 64), (256, 4, 2, 16)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_a_large_query_element_takes_no_bits_from_the_others(ctx, ops, dev, dtype, wide, hd, heads, n_kv, page_rows):
    """Where a channel of the keys is zero, what the query has there makes no difference, however large it is; one head has ordinary queries beside the others'."""
    pool = filled(90, [150, 500, 7], page_rows, n_kv, hd, dtype)
    pool.planes[0, ..., 5] = 0
    pool.max_pages += 2048 // page_rows if wide else 0
    d, q = OnDevice(dev, pool), normal(91, 3, heads, hd)
    for large in (0.0, 2.0 ** 12, 2.0 ** 19, 2.0 ** 24, 2.0 ** 40, 2.0 ** 100, 3e38):
        q[:, 1:, 5] = large
        got, want = attend(ctx, ops, dev, d, q), pool.attention(q)
        for h in range(heads):
            assert_f32_parity(got[:, h], want[:, h], f"{large}, head {h}")


@pytest.mark.parametrize("bits", [4, 20, 30, 40, 60])
@pytest.mark.parametrize("hd,heads,n_kv,page_rows", [(64, 8, 2, 16), (32, 3, 3, 32), (128, 8, 1, 64), (256, 4, 2, 16)])
@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_values_that_light_rows_alone_hold(ctx, ops, dev, dtype, hd, heads, n_kv, page_rows, bits):
    """One row draws nearly all weight and holds zeros in half of the channels; the others' weights are 2^-bits of it and are all that these channels have.
    An exponent of at most bits + 2 in magnitude is rounded at most eight times (square root, its inverse, log2(e), their product, the product with q, k's sum, the largest taken off), and
    exp2 is off by less than 2^-22, two halves of a weight by 2^-19: a weight by (8 ln2 (bits + 2) + 4 + 32) 2^-24 of itself.  Sums of n rows in f32 add n 2^-24 in whatever
    order, the joins a few more."""
    n = 61
    pool = filled(92, [n, 1], page_rows, n_kv, hd, dtype)
    pool.max_pages += 2048 // page_rows if bits % 20 == 0 else 0
    q = np.zeros((2, heads, hd), np.float32)
    q[..., 3] = 64.0
    for i, page in enumerate(pool.held[0]):  # row r's exponent: a multiple of 2^-3 about `bits` below row 33's
        pool.planes[0, page] = 0
        for r in range(page_rows):
            x = bits + (i * page_rows + r) % 9 / 8 if i * page_rows + r != 33 else 0.0
            pool.planes[0, page, :, r, 3] = np.round(-x * np.log(2) * np.sqrt(hd) / 64 * 1024) / 1024
    page, r = pool.held[0][33 // page_rows], 33 % page_rows
    pool.planes[1, page, :, r, :hd // 2] = 0
    got, want = attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q)
    magnitude = R.Pool.attention(_absolute(pool), q)
    steps = 8 * np.log(2) * (bits + 2) + 4 + 32 + n + 8
    off = np.abs(got[0] - want[0]) / magnitude[0]
    assert off.max() <= steps * 2.0 ** -24, (off.max() * 2.0 ** 24, steps)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,page_rows", [(64, 8, 2, 16), (32, 3, 3, 32), (128, 8, 1, 64), (256, 4, 2, 16)])
@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_every_weight_keeps_its_bits(ctx, ops, dev, dtype, wide, hd, heads, n_kv, page_rows):
    """Values of which each row has one, in a channel of its own, under weights from 1 down to 2^-90 in any order: outputs are the weights themselves.  As above but for the
    sums: a channel has one term, the weights' sum is 1 to 3 and of few that matter."""
    pool = filled(94, [hd], page_rows, n_kv, hd, dtype)
    pool.max_pages += 2048 // page_rows if wide else 0
    q = np.zeros((1, heads, hd), np.float32)
    q[..., 3] = 64.0
    octaves = np.random.default_rng(95).permutation(hd) * (90 / hd)
    keys = np.round(-octaves * np.log(2) * np.sqrt(hd) / 64 * 64) / 64
    for i, page in enumerate(pool.held[0]):
        pool.planes[:, page] = 0
        for r in range(min(page_rows, hd - i * page_rows)):
            pool.planes[0, page, :, r, 3] = keys[i * page_rows + r]
            pool.planes[1, page, :, r, i * page_rows + r] = 1 + r / 64
    got, want = attend(ctx, ops, dev, OnDevice(dev, pool), q)[0], pool.attention(q)[0]
    steps = 8 * np.log(2) * (octaves + 3) + 4 + 32 + 64
    assert np.all(np.abs(got - want) <= steps * 2.0 ** -24 * want), (np.abs(got / want - 1) * 2.0 ** 24 / steps).max()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,page_rows", [(64, 8, 2, 16), (32, 3, 3, 32), (128, 8, 1, 64), (256, 4, 2, 16), (64, 34, 2, 32)])
@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
def test_queries_as_small_as_keys_are_large(ctx, ops, dev, dtype, wide, hd, heads, n_kv, page_rows):
    """Channels whose keys are 2^28 times as large as others', and their queries as small: all of them make the scores alike.  Some heads have but one such element, some none."""
    lens = [300, 40]
    pool = filled(96, lens, page_rows, n_kv, hd, dtype)
    pool.max_pages += 2048 // page_rows if wide else 0
    e = np.random.default_rng(97).integers(0, 29, hd)
    x = np.clip(np.random.default_rng(98).standard_normal(pool.planes[0].shape), -3.99, 3.99)  # (times 2^14 an f16)
    pool.planes[0] = np.where(np.isnan(pool.planes[0]), np.nan, x * 2.0 ** (e - 14)).astype(R.TYPES[dtype])
    q = (normal(99, 2, heads, hd) * 2.0 ** (14 - e)).astype(np.float32)
    one = int(np.argmax(e))
    if heads > 4:
        q[:, 1] = np.where(np.arange(hd) == one, q[:, 1], np.where(e == e.min(), q[:, 1], 0))
        q[:, 2] = np.where(e <= e.min() + 3, q[:, 2], 0)
    got, want = attend(ctx, ops, dev, OnDevice(dev, pool), q), pool.attention(q)
    for s in range(2):
        for h in range(heads):
            assert_f32_parity(got[s, h], want[s, h], f"sequence {s}, head {h}")


def _absolute(pool):
    """The pool with its values' magnitudes."""
    p = R.Pool(pool.S, pool.max_pages, pool.n_pages, pool.R, pool.n_kv, pool.hd, pool.dtype)
    p.held, p.lens, p.planes = pool.held, pool.lens, pool.planes.copy()
    p.planes[1] = np.abs(p.planes[1])
    return p


@pytest.mark.parametrize("seqs,n_pages", [(40, 50), (300, 400), (4096, 8400)])
def test_moves_of_a_reservation_are_in_the_sequences_order(ops, dev, seqs, n_pages):
    """Many that write to a few shared pages: the list is the lists' own, move by move, in every run."""
    rng = np.random.default_rng(seqs)
    parents = [0, 1, 2] + [int(p) for p in rng.integers(0, 3, seqs - 3)]
    counts = [int(c) for c in rng.integers(0, 3, seqs)]
    for _ in range(3):
        pool = R.Pool(seqs, 4, n_pages, 16, 1, 32, KV_F16, n_planes=1)
        pool.reserve([20, 7, 33] + [0] * (seqs - 3))
        pool.fork(parents)
        d = OnDevice(dev, pool)
        start, moves = dev(np.zeros(seqs, np.uint32)), dev(np.zeros(kv_pages_moves_words(d.pages), np.uint32))
        want = pool.reserve(counts)
        ops.kv_pages_reserve(d.pages, dev(u32(*counts)), start, moves)
        assert want[2] == 0 and len(want[1]) > seqs // 2
        assert moves_of(moves) == (want[1], 0)
        assert np.array_equal(start.download(np.uint32, seqs), u32(*want[0]))
        d.check(planes=False)


@pytest.mark.parametrize("dtype", [KV_F32, KV_F16])
@pytest.mark.parametrize("hd,heads,n_kv,page_rows,lens", ATTENTION[2:20:3])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_in_place_of_its_queries(ctx, ops, dev, wide, hd, heads, n_kv, page_rows, lens, dtype):
    """In one launch, over shares and joined: the same bits as into an array of its own."""
    pool = filled(len(lens) + hd, lens, page_rows, n_kv, hd, dtype)
    pool.max_pages += 2048 // page_rows if wide else 0
    d, q = OnDevice(dev, pool), normal(11, len(lens), heads, hd) * np.float32(1.5)
    want = attend(ctx, ops, dev, d, q)
    d_q, width = dev(q), heads * hd
    scratch = dev(np.full(attention_paged_scratch_floats(len(lens), heads, n_kv, hd), np.nan, np.float32))
    ops.encode_attention_paged(d.pages, d_q, width, d.plane(0), d.plane(1), dtype, d_q, width, scratch, heads, n_kv, hd)
    assert np.array_equal(back(d_q, q), want)
