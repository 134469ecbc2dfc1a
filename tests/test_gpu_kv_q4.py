"""The KV cache held in 4 bits on the GPU against its numpy form (kv_q4_ref.py): rows appended and read back bit for bit, attention of
one token and of a prompt within the bar of f32 outputs (the quantized values are exact operands; products and sums keep f32's
bits), what rows have gathered, and the eviction, which moves bytes."""
import numpy as np
import pytest

import kv_q4_ref as R
import wick_amd as W
from conftest import assert_f32_parity
from wick_amd.lfm2 import Lfm2Ops, attention_q4_scratch_floats, kv_q4_bytes, kv_q4_evict_scratch_floats, rope_theta_scale

pytestmark = pytest.mark.gpu


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


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def filled(seed, max_seq, n_kv, hd, used):
    """Caches of normal keys and values whose rows from `used` on hold NaN."""
    k, v = R.Cache(max_seq, n_kv, hd), R.Cache(max_seq, n_kv, hd)
    k.append(0, normal(seed, used, n_kv, hd)), v.append(0, normal(seed + 1, used, n_kv, hd))
    return k, v


def scratch_for(ctx, dev, *args, **kw):
    n = attention_q4_scratch_floats(*args, **kw)
    return dev(np.full(max(n, 4), np.nan, np.float32))  # (contents need not be kept, nor be anything)


# ---- append, read back ------------------------------------------------------------------------

def special_blocks():
    """Blocks at the rule's borders: zeros, a scale that rounds to 0 or to the smallest half, the largest value and one beyond it, values
    that are none, magnitudes of both signs, one value alone, halves between two steps."""
    b = normal(3, 16, 32)
    b[0] = 0
    b[1], b[2] = b[1] * 1e-8, 0
    b[2, 5] = 2.0 ** -22  # d = 2^-25: rounds to 0
    b[3], b[3, 9] = 0, 2.0 ** -21
    b[4, 0], b[5, 31], b[5, 30] = 65504.0, -65504.0, 1.0
    b[6, 7], b[7, 3], b[8, 0], b[9, 31] = 65520.0, np.inf, np.nan, -np.inf
    b[10, 4], b[10, 20] = 5.0, -5.0
    b[11], b[11, 17] = 0, -3.0
    b[12] = np.arange(32) / 4.0 - 4.0
    b[13] = -b[12]
    b[14] = np.float32(1e-40)
    b[15] = -0.0
    return b


@pytest.mark.parametrize("hd,n_kv,n,row,extra", [(64, 8, 1, 700, 0), (64, 8, 37, 0, 4), (32, 1, 5, 3, 0), (128, 3, 9, 100, 64), (256, 2, 33, 7, 12), (64, 2, 300, 211, 0)])
def test_append_and_read_back(ctx, ops, dev, hd, n_kv, n, row, extra):
    max_seq, stride = row + n + 5, n_kv * hd + extra
    k, v = normal(n, n, stride), normal(n + 1, n, stride) * 3
    special = special_blocks().ravel()
    k[:, :n_kv * hd].reshape(n, -1)[0, :min(n_kv * hd, special.size)] = special[:n_kv * hd]
    v[n - 1, :min(n_kv * hd, special.size)] = special[::-1][:n_kv * hd]
    refs, caches = [R.Cache(max_seq, n_kv, hd, fill=0xa5) for _ in range(2)], []
    for ref, x in zip(refs, (k, v)):
        caches.append(dev(ref.raw))
        ref.append(row, x[:, :n_kv * hd].reshape(n, n_kv, hd))
    assert kv_q4_bytes(max_seq, n_kv, hd) == refs[0].raw.size
    ops.encode_kv_q4_append(dev(k), dev(v), stride, *caches, row, n, max_seq, n_kv, hd)
    for ref, cache in zip(refs, caches):
        assert np.array_equal(ref.words, (got := back(cache, ref.raw))[:ref.words.size * 4].view(np.uint32).reshape(ref.words.shape))
        a, b = ref.raw[ref.words.size * 4:].view(np.float16), got[ref.words.size * 4:].view(np.float16)
        assert np.array_equal(a, b, equal_nan=True)
        assert np.array_equal(np.signbit(a[a == 0]), np.signbit(b[a == 0]))
        out = np.full((n, stride), 7.0, np.float32)
        d_out = dev(out)
        ops.encode_kv_q4_read(cache, d_out, stride, row, n, max_seq, n_kv, hd)
        out = back(d_out, out)
        want = ref.values(row, n).transpose(1, 0, 2).reshape(n, -1).astype(np.float32)  # (exact: four bits times eleven)
        assert np.array_equal(out[:, :n_kv * hd], want, equal_nan=True) and np.all(out[:, n_kv * hd:] == 7.0)


def test_append_at_a_row_on_the_device(ctx, ops, dev):
    """The row from device memory wins over the by-value one; rows past the cache are dropped."""
    max_seq, n_kv, hd, n = 20, 2, 64, 6
    x = normal(1, n, n_kv, hd)
    for row in (0, 9, 14, 16, 19, 20, 4000000000, 4294967295):
        ref = R.Cache(max_seq, n_kv, hd)
        a, b = dev(ref.raw), dev(ref.raw)
        if row < max_seq:
            ref.append(row, x)
        ops.encode_kv_q4_append(dev(x), dev(x), n_kv * hd, a, b, 0, n, max_seq, n_kv, hd, d_row=dev(np.array([row], np.uint32)))
        assert np.array_equal(back(a, ref.raw), ref.raw) and np.array_equal(back(b, ref.raw), ref.raw)


# ---- attention of one token ---------------------------------------------------------------------

DECODE = [  # head_dim, heads, KV heads, rows in use, rows
    (64, 16, 8, 1, 64), (64, 16, 8, 2, 64), (64, 16, 8, 31, 256), (64, 32, 8, 64, 64), (64, 16, 8, 65, 4096), (64, 8, 8, 257, 300),
    (64, 24, 3, 1000, 1001), (64, 16, 8, 4097, 8192), (64, 64, 1, 700, 700), (64, 5, 5, 2049, 40000), (64, 34, 2, 300, 512),
    (32, 4, 2, 77, 100), (32, 8, 1, 5000, 5000), (128, 8, 2, 129, 4096), (128, 32, 8, 3001, 3001), (256, 4, 1, 33, 64), (256, 6, 2, 2500, 2600),
    (32, 80, 1, 170000, 180000), (32, 66000, 33000, 2, 2),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,seq,max_seq", DECODE)
def test_attention_of_one_token(ctx, ops, dev, hd, heads, n_kv, seq, max_seq, weights):
    k, v = filled(seq, max_seq, n_kv, hd, seq)
    q = 2 * normal(seq + 5, 1, heads, hd)
    out, p = R.attention(q, k, v, seq - 1)
    scratch = scratch_for(ctx, dev, 1, max_seq, heads, n_kv, hd, weights)
    d_out, w0 = dev(np.full(heads * hd, np.nan, np.float32)), np.abs(normal(9, n_kv, max_seq))
    d_w, d_k, d_v, d_q = dev(w0), dev(k.raw), dev(v.raw), dev(q)
    for d_pos in (None, dev(np.array([seq - 1], np.uint32))):  # by value, from device memory
        ops.encode_attention_q4(d_q, d_k, d_v, d_out, scratch, seq if d_pos is None else 0, max_seq, heads, n_kv, hd, weights=d_w if weights else None, d_pos=d_pos)
        assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), out[0], f"d_pos {d_pos}")
        if weights:
            w0[:, :seq] += R.gathered(p, n_kv)
            got = back(d_w, w0)
            assert_f32_parity(got[:, :seq], w0[:, :seq], "weights")
            assert np.array_equal(got[:, seq:], w0[:, seq:])
            w0 = got
        else:
            assert np.array_equal(back(d_w, w0), w0)


def test_attention_over_no_row_and_past_the_cache(ctx, ops, dev):
    hd, heads, n_kv, max_seq = 64, 4, 2, 96
    k, v = filled(1, max_seq, n_kv, hd, max_seq)
    q = normal(2, 1, heads, hd)
    scratch, d_out, w0 = scratch_for(ctx, dev, 1, max_seq, heads, n_kv, hd, True), dev(np.full(heads * hd, np.nan, np.float32)), np.zeros((n_kv, max_seq), np.float32)
    d_w = dev(w0)
    ops.encode_attention_q4(dev(q), dev(k.raw), dev(v.raw), d_out, scratch, 0, max_seq, heads, n_kv, hd, weights=d_w)
    assert np.array_equal(d_out.download(np.float32, heads * hd), np.zeros(heads * hd, np.float32)) and not back(d_w, w0).any()
    for pos in (max_seq - 1, max_seq, 4294967295):  # a position past the cache sees all of it
        ops.encode_attention_q4(dev(q), dev(k.raw), dev(v.raw), d_out, scratch, 0, max_seq, heads, n_kv, hd, d_pos=dev(np.array([pos], np.uint32)))
        assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), R.attention(q, k, v, max_seq - 1)[0][0], f"{pos}")


# ---- attention of a prompt -----------------------------------------------------------------------

PROMPTS = [  # head_dim, heads, KV heads, first row, tokens, rows behind them, floats between tokens
    (64, 16, 8, 0, 1, 0, 0), (64, 16, 8, 0, 2, 9, 4), (64, 16, 8, 700, 23, 5, 0), (64, 16, 8, 0, 64, 0, 64), (64, 32, 8, 0, 65, 1, 0),
    (64, 16, 8, 0, 555, 200, 0), (64, 16, 8, 63, 129, 0, 0), (64, 3, 3, 1000, 40, 24, 0), (64, 7, 1, 130, 33, 3, 4), (64, 24, 3, 5, 200, 0, 0), (64, 40, 1, 77, 17, 2, 0),
    (64, 8, 4, 3000, 300, 0, 0),
    (32, 4, 2, 10, 100, 4, 0), (32, 6, 1, 500, 9, 0, 0), (128, 8, 2, 100, 150, 7, 8), (128, 4, 4, 0, 257, 0, 0), (128, 8, 1, 2000, 5, 0, 0),
    (256, 4, 2, 33, 70, 0, 0), (256, 2, 1, 900, 130, 30, 12), (256, 8, 1, 0, 3, 0, 0),
]


LARGE = [  # more than 64 rows of a KV head, and up to and beyond 12 million pairs of a query and a key: the tiled kernels, split over few and many workgroups, one and two a CU
    (64, 16, 4, 1777, 333, 0, 0), (64, 32, 8, 0, 1030, 3, 0), (64, 2, 1, 66000, 65, 0, 0), (64, 12, 4, 900, 701, 5, 4), (128, 6, 2, 2222, 301, 0, 8),
    (128, 16, 4, 7, 2050, 0, 0), (256, 3, 1, 1300, 500, 40, 0), (32, 8, 8, 1000, 1500, 0, 0), (32, 24, 2, 20001, 67, 0, 0),
    (64, 16, 4, 1777, 430, 2, 0), (64, 2, 1, 100000, 65, 0, 0), (64, 12, 4, 1300, 701, 5, 4), (128, 6, 2, 3333, 601, 0, 8), (256, 3, 1, 4400, 901, 0, 0),
]


@pytest.mark.parametrize("hd,heads,n_kv,pos0,n,behind,pad,weights", [(*p, w) for p in PROMPTS for w in (False, True)] + [(*p, True) for p in LARGE])
def test_attention_of_a_prompt(ctx, ops, dev, hd, heads, n_kv, pos0, n, behind, pad, weights):
    max_seq, stride = pos0 + n + behind, heads * hd + pad
    k, v = filled(n, max_seq, n_kv, hd, pos0 + n)
    q = 2 * normal(n + 5, n, stride)
    ref, p = R.attention(q[:, :heads * hd].reshape(n, heads, hd), k, v, pos0)
    scratch = scratch_for(ctx, dev, n, max_seq, heads, n_kv, hd, weights)
    out, w0 = np.full((n + 1, stride), 7.0, np.float32), np.abs(normal(9, n_kv, max_seq))
    d_out, d_w = dev(out), dev(w0)
    ops.encode_attention_prefill_q4(dev(q), stride, dev(k.raw), dev(v.raw), d_out, stride, scratch, pos0, n, max_seq, heads, n_kv, hd, weights=d_w if weights else None)
    out = back(d_out, out)
    assert_f32_parity(out[:n, :heads * hd].reshape(n, heads, hd), ref, "out")
    for j in (0, n // 2, n - 1):  # (and of tokens on their own: the first ones of a prompt weigh little in the sum over all)
        assert_f32_parity(out[j, :heads * hd].reshape(heads, hd), ref[j], f"token {j}")
    assert np.all(out[n] == 7.0) and np.all(out[:, heads * hd:] == 7.0)  # nothing between the tokens or behind the last one
    got = back(d_w, w0)
    if weights:
        w0[:, :pos0 + n] += R.gathered(p, n_kv)
        assert_f32_parity(got[:, :pos0 + n], w0[:, :pos0 + n], "weights")
        assert np.array_equal(got[:, pos0 + n:], w0[:, pos0 + n:])
    else:
        assert np.array_equal(got, w0)


@pytest.mark.parametrize("hd,heads,n_kv,pos0,n", [(64, 4, 2, 0, 100), (128, 2, 1, 70, 30), (64, 4, 2, 300, 1), (32, 2, 2, 5, 60), (256, 2, 2, 5, 60),
                                                  (64, 8, 2, 1500, 600), (128, 8, 4, 700, 600), (32, 16, 2, 300, 1200), (256, 4, 2, 500, 700),
                                                  (64, 16, 2, 1500, 600), (128, 16, 4, 1000, 700), (256, 8, 2, 1700, 800)])
def test_a_row_held_as_nan_is_seen_by_those_that_see_it(ctx, ops, dev, hd, heads, n_kv, pos0, n):
    """Of keys in head 0, of values in the last head: NaN to the tokens from that row on, everything as without it to those before."""
    max_seq, bad = pos0 + n, pos0 + n // 2
    k, v = filled(n, max_seq, n_kv, hd, max_seq)
    q = normal(4, n, heads, hd)
    clean, p = R.attention(q, k, v, pos0)
    k.scales[0, bad, 0], v.scales[n_kv - 1, bad, hd // 32 - 1] = np.nan, np.inf
    group, hit = heads // n_kv, np.zeros((n, heads), bool)
    hit[bad - pos0:, :group] = hit[bad - pos0:, heads - group:] = True
    scratch, d_out, d_w = scratch_for(ctx, dev, n, max_seq, heads, n_kv, hd, True), dev(np.zeros((n, heads, hd), np.float32)), dev(np.zeros((n_kv, max_seq), np.float32))
    d_k, d_v, d_q = dev(k.raw), dev(v.raw), dev(q)
    if n == 1:
        ops.encode_attention_q4(d_q, d_k, d_v, d_out, scratch, max_seq, max_seq, heads, n_kv, hd, weights=d_w)
    else:
        ops.encode_attention_prefill_q4(d_q, heads * hd, d_k, d_v, d_out, heads * hd, scratch, pos0, n, max_seq, heads, n_kv, hd, weights=d_w)
    out = d_out.download(np.float32, n * heads * hd).reshape(n, heads, hd)
    assert np.isnan(out[hit]).all()
    if not hit.all():
        assert_f32_parity(out[~hit], clean[~hit], "tokens that do not see it")
    got = d_w.download(np.float32, n_kv * max_seq).reshape(n_kv, max_seq)
    assert np.isnan(got[[0, n_kv - 1]]).all()  # (the last token sees every row)
    assert_f32_parity(got[1:n_kv - 1], R.gathered(p, n_kv)[1:n_kv - 1], "weights of the other heads") if n_kv > 2 else None


@pytest.mark.parametrize("heads,n_kv,seq,n", [(4, 2, 300, 20), (16, 4, 1200, 700), (16, 4, 1600, 900)])
@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1e4, 3e4])
def test_queries_of_all_sizes(ctx, ops, dev, factor, heads, n_kv, seq, n):
    """Tiny queries weigh all rows alike, huge ones one row alone; both with keys that answer in kind."""
    hd = 64
    k, v = R.Cache(seq, n_kv, hd), R.Cache(seq, n_kv, hd)
    k.append(0, normal(1, seq, n_kv, hd) * np.float32(1 / factor if factor > 1 else 1000)), v.append(0, normal(2, seq, n_kv, hd) * np.float32(1e-4))
    q = (normal(3, n, heads, hd) * factor).astype(np.float32)
    scratch, d_out = scratch_for(ctx, dev, n, seq, heads, n_kv, hd), dev(np.zeros((n, heads, hd), np.float32))
    ops.encode_attention_prefill_q4(dev(q), heads * hd, dev(k.raw), dev(v.raw), d_out, heads * hd, scratch, seq - n, n, seq, heads, n_kv, hd)
    assert_f32_parity(d_out.download(np.float32, q.size).reshape(q.shape), R.attention(q, k, v, seq - n)[0], "out")
    ops.encode_attention_q4(dev(q[n - 1]), dev(k.raw), dev(v.raw), d_out, scratch, seq, seq, heads, n_kv, hd)
    assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), R.attention(q[n - 1:], k, v, seq - 1)[0][0], "one token")


@pytest.mark.parametrize("hd,heads,n_kv,n", [(64, 4, 2, 50), (128, 8, 2, 1100), (128, 16, 2, 1400)])
def test_a_value_that_is_not_finite_stays_with_its_query(ctx, ops, dev, hd, heads, n_kv, n):
    k, v = filled(1, n, n_kv, hd, n)
    q = normal(3, n, heads, hd)
    ref = R.attention(q, k, v, 0)[0]
    q[10, 1, 5], q[n - 20, 2, 60] = np.nan, np.inf
    scratch, d_out = scratch_for(ctx, dev, n, n, heads, n_kv, hd), dev(np.zeros((n, heads, hd), np.float32))
    ops.encode_attention_prefill_q4(dev(q), heads * hd, dev(k.raw), dev(v.raw), d_out, heads * hd, scratch, 0, n, n, heads, n_kv, hd)
    out, hit = d_out.download(np.float32, q.size).reshape(q.shape), np.zeros((n, heads), bool)
    hit[10, 1] = hit[n - 20, 2] = True
    assert np.isnan(out[hit]).all()
    assert_f32_parity(out[~hit], ref[~hit], "the others")


def test_heads_past_four_gigabytes(ctx, ops, dev):
    """Caches whose last head starts behind 2^32 bytes: append, both forms of attention, eviction and read at its rows."""
    hd, heads, n_kv, used, n = 256, 8, 8, 200, 20
    max_seq = (1 << 32) // (hd // 2) // 7 + 1000
    size = kv_q4_bytes(max_seq, n_kv, hd)
    assert size > 1 << 32
    big = [ctx.alloc(size) for _ in range(2)]
    small = [R.Cache(used, n_kv, hd) for _ in range(2)]
    xs = [normal(i, used, n_kv, hd) for i in range(2)]
    for s, x in zip(small, xs):
        s.append(0, x)
    ops.encode_kv_q4_append(dev(xs[0]), dev(xs[1]), n_kv * hd, *big, 0, used, max_seq, n_kv, hd)
    q = normal(5, n, heads, hd)
    w = ctx.alloc(4 * n_kv * max_seq)
    for c in range(n_kv):
        w.upload(np.zeros(used, np.float32), 4 * c * max_seq)
    scratch, d_out = scratch_for(ctx, dev, n, max_seq, heads, n_kv, hd, True), dev(np.zeros((n, heads, hd), np.float32))
    ref, p = R.attention(q, *small, used - n)
    ops.encode_attention_prefill_q4(dev(q), heads * hd, *big, d_out, heads * hd, scratch, used - n, n, max_seq, heads, n_kv, hd, weights=w)
    assert_f32_parity(d_out.download(np.float32, q.size).reshape(q.shape), ref, "prompt")
    ops.encode_attention_q4(dev(q[n - 1]), *big, d_out, scratch, used, max_seq, heads, n_kv, hd)
    assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), ref[n - 1], "one token")
    kept, drop = dev(np.zeros((n_kv, used - 50), np.uint32)), 50
    got_w = np.stack([w.download(np.float32, used, 4 * c * max_seq) for c in range(n_kv)])
    assert_f32_parity(got_w, R.gathered(p, n_kv), "weights")
    ops.encode_kv_q4_evict(*big, w, kept, dev(np.zeros(max(4, kv_q4_evict_scratch_floats(used, n_kv)), np.float32)), used, 2, 10, drop, max_seq, n_kv, hd)
    rows = kept.download(np.uint32, n_kv * (used - drop)).reshape(n_kv, -1)
    d_back = dev(np.zeros((used - drop, n_kv, hd), np.float32))
    for s, b in zip(small, big):
        ops.encode_kv_q4_read(b, d_back, n_kv * hd, 0, used - drop, max_seq, n_kv, hd)
        got = d_back.download(np.float32, (used - drop) * n_kv * hd).reshape(used - drop, n_kv, hd)
        for c in range(n_kv):
            assert np.array_equal(rows[c], R.evicted(got_w[c], used, 2, 10, drop))
            assert np.array_equal(got[:, c], s.values(0, used)[c][rows[c]].astype(np.float32))
    w.free()
    for b in big:
        b.free()


# ---- eviction ------------------------------------------------------------------------------------

EVICT = [  # head_dim, KV heads, rows in use, rows, kept first, kept last, dropped
    (64, 8, 300, 400, 4, 32, 100), (64, 2, 1, 1, 0, 0, 1), (64, 1, 50, 50, 0, 0, 50), (64, 3, 50, 64, 10, 39, 1), (64, 8, 3000, 3000, 64, 256, 800),
    (32, 2, 1025, 1100, 0, 0, 1), (32, 1, 2500, 2500, 1, 1, 2498), (128, 2, 1024, 1024, 7, 100, 333), (256, 1, 700, 701, 0, 650, 50), (256, 2, 1500, 1600, 1400, 0, 60),
    (64, 1, 9000, 9000, 4, 1000, 5), (32, 1, 40000, 40000, 0, 0, 20000), (32, 2, 150000, 150001, 5, 77, 60000), (128, 1, 4096, 4096, 0, 0, 4096), (64, 1, 4097, 5000, 4090, 0, 7),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
@pytest.mark.parametrize("hd,n_kv,seq,max_seq,keep,recent,drop", EVICT)
def test_evict(ctx, ops, dev, hd, n_kv, seq, max_seq, keep, recent, drop, kind):
    rng = np.random.default_rng(seq + drop)
    w = np.exp(2 * rng.standard_normal((n_kv, max_seq))).astype(np.float32)
    if kind == "ties":  # few different values, and none at all
        w = np.floor(w * 2) / 4 * (rng.random(w.shape) > 0.3)
    if kind == "special":
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.2] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
        w[rng.random(w.shape) < 0.2] = -0.0
        w[rng.random(w.shape) < 0.2] = 0.0
        w[rng.random(w.shape) < 0.2] *= -1
    w = w.astype(np.float32)
    caches = [R.Cache(max_seq, n_kv, hd) for _ in range(2)]
    for c in caches:
        c.raw[:] = rng.integers(0, 256, c.raw.size, np.uint8)  # bytes are moved, whatever they stand for
    left = seq - drop
    d_caches, d_w, d_kept = [dev(c.raw) for c in caches], dev(w), dev(np.full((n_kv, left + 1), 9, np.uint32))
    scratch = dev(np.full(max(4, kv_q4_evict_scratch_floats(seq, n_kv)), np.nan, np.float32))
    ops.encode_kv_q4_evict(*d_caches, d_w, d_kept, scratch, seq, keep, recent, drop, max_seq, n_kv, hd)
    want = np.stack([R.evicted(w[c], seq, keep, recent, drop) for c in range(n_kv)]).reshape(n_kv, left)
    got = d_kept.download(np.uint32, n_kv * left + 1)
    assert np.array_equal(got[:-1].reshape(n_kv, left), want) and got[-1] == 9
    w_after = w.copy()
    for c in range(n_kv):
        w_after[c, :left], w_after[c, left:seq] = w[c, want[c]], 0
        for cache in caches:
            cache.words[c, :left], cache.scales[c, :left] = cache.words[c, want[c]], cache.scales[c, want[c]]
    assert np.array_equal(back(d_w, w).view(np.uint32), w_after.view(np.uint32))
    for cache, d in zip(caches, d_caches):
        assert np.array_equal(back(d, cache.raw), cache.raw)


# ---- together --------------------------------------------------------------------------------------

def test_a_captured_step_replayed_while_the_position_moves(ctx, ops, dev):
    """Append and attention, weights gathered, in one graph, the row and position from device memory; eager work between replays.
    Every replay against f64."""
    hd, heads, n_kv, max_seq, start, steps = 64, 8, 4, 700, 250, 12
    k, v = filled(1, max_seq, n_kv, hd, start)
    d_k, d_v, d_w = dev(k.raw), dev(v.raw), dev(np.zeros((n_kv, max_seq), np.float32))
    x, d_x = normal(4, steps, 3, heads * hd), dev(np.zeros((3, heads * hd), np.float32))
    d_q, d_kx, d_vx = d_x.ptr, d_x.ptr + 4 * heads * hd, d_x.ptr + 8 * heads * hd
    d_pos, d_out, scratch = dev(np.zeros(1, np.uint32)), dev(np.zeros(heads * hd, np.float32)), scratch_for(ctx, dev, 1, max_seq, heads, n_kv, hd, True)
    ctx.sync()
    ctx.graph_begin()
    ops.encode_kv_q4_append(d_kx, d_vx, heads * hd, d_k, d_v, 0, 1, max_seq, n_kv, hd, d_row=d_pos)
    ops.encode_attention_q4(d_q, d_k, d_v, d_out, scratch, 0, max_seq, heads, n_kv, hd, weights=d_w, d_pos=d_pos)
    g = ctx.graph_end()
    total = np.zeros((n_kv, max_seq))
    for s in range(steps):
        pos = start + s if s < steps - 1 else 699  # the last one on the cache's last row, over rows that hold NaN until they are written
        if pos == 699:
            fill = normal(8, 699 - (start + s), n_kv, hd)
            ops.encode_kv_q4_append(dev(fill), dev(fill), n_kv * hd, d_k, d_v, start + s, len(fill), max_seq, n_kv, hd)  # eager, between replays
            k.append(start + s, fill), v.append(start + s, fill)
        d_x.upload(x[s]), d_pos.upload(np.array([pos], np.uint32))
        ctx.graph_launch(g)
        k.append(pos, x[s, 1, :n_kv * hd].reshape(1, n_kv, hd)), v.append(pos, x[s, 2, :n_kv * hd].reshape(1, n_kv, hd))
        ref, p = R.attention(x[s, 0].reshape(1, heads, hd), k, v, pos)
        total[:, :pos + 1] += R.gathered(p, n_kv)
        assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), ref[0], f"step {s}")
        assert_f32_parity(d_w.download(np.float32, n_kv * max_seq).reshape(n_kv, -1), total, f"weights of step {s}")
    ctx.graph_destroy(g)


def random_cache(rng, max_seq, n_kv, hd):
    c = R.Cache(max_seq, n_kv, hd)
    c.raw[:] = rng.integers(0, 256, c.raw.size, np.uint8)
    return c


def assert_evicted(got, before, w, d_w, d_kept, seq, keep, recent, drop):
    """Caches (device) and weights behind an eviction from `before` (host) by weights w."""
    n_kv, left = w.shape[0], seq - drop
    kept = d_kept.download(np.uint32, n_kv * left).reshape(n_kv, left)
    w_after = w.copy()
    for c in range(n_kv):
        assert np.array_equal(kept[c], R.evicted(w[c], seq, keep, recent, drop))
        w_after[c, :left], w_after[c, left:seq] = w[c, kept[c]], 0
        for cache in before:
            cache.words[c, :left], cache.scales[c, :left] = cache.words[c, kept[c]], cache.scales[c, kept[c]]
    assert np.array_equal(back(d_w, w), w_after)
    for cache, d in zip(before, got):
        assert np.array_equal(back(d, cache.raw), cache.raw)


@pytest.mark.parametrize("hd,n_kv,seq,drop", [(64, 3, 9000, 2500), (256, 1, 3000, 700), (32, 2, 4097, 4000)])
def test_a_captured_eviction_replayed(ctx, ops, dev, hd, n_kv, seq, drop):
    """Its counters and histograms are as it needs them in every replay, with other evictions over the same scratch between."""
    rng, max_seq, keep, recent = np.random.default_rng(seq), seq + 30, 8, 64
    small = kv_q4_evict_scratch_floats(500, n_kv)
    scratch = dev(np.full(max(small, kv_q4_evict_scratch_floats(seq, n_kv)), np.nan, np.float32))
    d_caches, d_w = [dev(random_cache(rng, max_seq, n_kv, hd).raw) for _ in range(2)], dev(np.zeros((n_kv, max_seq), np.float32))
    d_kept = dev(np.zeros((n_kv, seq), np.uint32))
    ctx.sync()
    ctx.graph_begin()
    ops.encode_kv_q4_evict(*d_caches, d_w, d_kept, scratch, seq, keep, recent, drop, max_seq, n_kv, hd)
    g = ctx.graph_end()
    for _ in range(4):
        caches, w = [random_cache(rng, max_seq, n_kv, hd) for _ in range(2)], rng.exponential(size=(n_kv, max_seq)).astype(np.float32)
        for d, c in zip([*d_caches, d_w], [*(c.raw for c in caches), w]):
            d.upload(c)
        ctx.graph_launch(g)
        assert_evicted(d_caches, caches, w, d_w, d_kept, seq, keep, recent, drop)
        w = back(d_w, w)
        ops.encode_kv_q4_evict(*d_caches, d_w, d_kept, scratch, 500, 3, 0, 120, max_seq, n_kv, hd)  # eager, between replays
        assert_evicted(d_caches, caches, w, d_w, d_kept, 500, 3, 0, 120)
    ctx.graph_destroy(g)


def test_two_evictions_at_once(ctx, ops, dev):
    """Two streams, each with caches and a scratch of its own."""
    rng, other = np.random.default_rng(1), W.RocmContext(0)
    hd, n_kv, seq, keep, recent, drop = 128, 4, 20000, 4, 100, 6000
    try:
        calls = []
        for o in (ops, Lfm2Ops(other)):
            caches, w = [random_cache(rng, seq, n_kv, hd) for _ in range(2)], rng.exponential(size=(n_kv, seq)).astype(np.float32)
            calls.append((o, caches, w, [dev(c.raw) for c in caches], dev(w), dev(np.zeros((n_kv, seq), np.uint32)), dev(np.zeros(kv_q4_evict_scratch_floats(seq, n_kv), np.float32))))
        ctx.sync()
        for o, _, _, d_caches, d_w, d_kept, scratch in calls:
            o.encode_kv_q4_evict(*d_caches, d_w, d_kept, scratch, seq, keep, recent, drop, seq, n_kv, hd)
        other.sync()
        for _, caches, w, d_caches, d_w, d_kept, _ in calls:
            assert_evicted(d_caches, caches, w, d_w, d_kept, seq, keep, recent, drop)
    finally:
        other.close()


@pytest.mark.parametrize("hd,heads,n_kv,n,pos0", [(64, 16, 4, 900, 700), (64, 16, 8, 70, 300), (128, 8, 2, 5, 4000)])
def test_a_captured_prompt_replayed(ctx, ops, dev, hd, heads, n_kv, n, pos0):
    """Bit for bit the eager call's output and weights, with other prompts over the same scratch between."""
    max_seq = pos0 + n
    k, v = filled(3, max_seq, n_kv, hd, max_seq)
    d_q, d_k, d_v, q = dev(np.zeros((n, heads * hd), np.float32)), dev(k.raw), dev(v.raw), normal(4, 3, n, heads * hd)
    scratch, d_out, d_w = scratch_for(ctx, dev, n, max_seq, heads, n_kv, hd, True), dev(np.zeros((n, heads * hd), np.float32)), dev(np.zeros((n_kv, max_seq), np.float32))

    def call(of):
        ops.encode_attention_prefill_q4(d_q, heads * hd, d_k, d_v, d_out, heads * hd, scratch, pos0, of, max_seq, heads, n_kv, hd, weights=d_w)

    def results():
        return d_out.download(np.uint32, n * heads * hd), d_w.download(np.uint32, n_kv * max_seq)

    ctx.sync()
    ctx.graph_begin()
    call(n)
    g = ctx.graph_end()
    for x in q:
        d_q.upload(x)
        got = []
        for run in (lambda: call(n), lambda: ctx.graph_launch(g), lambda: ctx.graph_launch(g)):
            d_w.upload(np.full((n_kv, max_seq), 0.25, np.float32))
            run()
            got.append(results())
            call(max(n // 3, 1))
        assert all(np.array_equal(a, b) for other in got[1:] for a, b in zip(got[0], other))
    ctx.graph_destroy(g)


@pytest.mark.parametrize("n,pos0", [(300, 500), (700, 500), (900, 700)])
def test_results_do_not_change_from_run_to_run(ctx, ops, dev, n, pos0):
    hd, heads, n_kv = 64, 16, 4
    k, v = filled(3, pos0 + n, n_kv, hd, pos0 + n)
    q, d_k, d_v = dev(normal(4, n, heads, hd)), dev(k.raw), dev(v.raw)
    scratch, got = scratch_for(ctx, dev, n, pos0 + n, heads, n_kv, hd, True), []
    for _ in range(3):
        d_out, d_w = dev(np.zeros((n, heads, hd), np.float32)), dev(np.zeros((n_kv, pos0 + n), np.float32))
        ops.encode_attention_prefill_q4(q, heads * hd, d_k, d_v, d_out, heads * hd, scratch, pos0, n, pos0 + n, heads, n_kv, hd, weights=d_w)
        ops.encode_attention_q4(q, d_k, d_v, d_out, scratch, pos0 + n, pos0 + n, heads, n_kv, hd, weights=d_w)
        got.append((d_out.download(np.uint32, n * heads * hd), d_w.download(np.uint32, n_kv * (pos0 + n))))
    assert all(np.array_equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


def test_two_contexts_at_once(ctx, ops, dev):
    """Two streams over the same caches, a scratch of its own each."""
    hd, heads, n_kv, seq = 64, 16, 8, 3000
    k, v = filled(3, seq, n_kv, hd, seq)
    q, d_k, d_v = normal(4, 2, heads, hd), dev(k.raw), dev(v.raw)
    other = W.RocmContext(0)
    try:
        ctx.sync()
        calls = []
        for i, o in enumerate((ops, Lfm2Ops(other))):
            calls.append((o, dev(q[i]), dev(np.zeros(heads * hd, np.float32)), scratch_for(ctx, dev, 1, seq, heads, n_kv, hd)))
        for _ in range(10):
            for o, d_q, d_out, scratch in calls:
                o.encode_attention_q4(d_q, d_k, d_v, d_out, scratch, seq, seq, heads, n_kv, hd)
        other.sync()
        for i, (_, _, d_out, _) in enumerate(calls):
            assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), R.attention(q[i:i + 1], k, v, seq - 1)[0][0], f"context {i}")
    finally:
        other.close()


def test_a_session_that_evicts(ctx, ops, dev):
    """A prompt, steps, an eviction, steps, another eviction: positions go on for the rotation, rows are counted anew, and what is
    appended behind an eviction starts with no weight."""
    hd, heads, n_kv, max_seq, eps = 64, 8, 4, 160, 1e-5
    theta = rope_theta_scale(hd, 1e6)
    rng = np.random.default_rng(5)
    d_norm = dev((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32))
    k, v = R.Cache(max_seq, n_kv, hd), R.Cache(max_seq, n_kv, hd)
    d_k, d_v, w = dev(k.raw), dev(v.raw), np.zeros((n_kv, max_seq), np.float32)
    d_w, none = dev(w), dev(np.zeros(1 << 16, np.float32))  # (f32 rows that nobody reads: the rotation's own append)
    scratch, d_out = scratch_for(ctx, dev, 128, max_seq, heads, n_kv, hd, True), dev(np.zeros((128, heads, hd), np.float32))
    pos = row = 0
    for n in (100, 1, 1, -60, 1, 70, -40, -10, 20, 1, 1):
        if n < 0:
            got_w, kept = back(d_w, w), dev(np.zeros((n_kv, row + n), np.uint32))
            ops.encode_kv_q4_evict(d_k, d_v, d_w, kept, dev(np.zeros(max(4, kv_q4_evict_scratch_floats(row, n_kv)), np.float32)), row, 4, 16, -n, max_seq, n_kv, hd)
            kept = kept.download(np.uint32, n_kv * (row + n)).reshape(n_kv, -1)
            for c in range(n_kv):
                assert np.array_equal(kept[c], R.evicted(got_w[c], row, 4, 16, -n))
                w[c, :row + n], w[c, row + n:row] = got_w[c, kept[c]], 0
                for cache in (k, v):
                    cache.words[c, :row + n], cache.scales[c, :row + n] = cache.words[c, kept[c]], cache.scales[c, kept[c]]
            row += n
            continue
        x = rng.standard_normal((3, n, heads * hd)).astype(np.float32)
        d_q, d_kx, d_vx = dev(x[0]), dev(x[1]), dev(x[2])
        ops.encode_qk_norm_rope_tokens(d_q, heads * hd, d_kx, d_vx, heads * hd, d_norm, d_norm, none, none, pos, n, pos + n, hd, heads, n_kv, eps, theta) \
            if (pos + n) * n_kv * hd <= 1 << 16 else pytest.fail("room")
        ops.encode_kv_q4_append(d_kx, d_vx, heads * hd, d_k, d_v, row, n, max_seq, n_kv, hd)
        q, kx = back(d_q, x[0]), back(d_kx, x[1])
        k.append(row, kx[:, :n_kv * hd].reshape(n, n_kv, hd)), v.append(row, x[2][:, :n_kv * hd].reshape(n, n_kv, hd))
        ref, p = R.attention(q.reshape(n, heads, hd), k, v, row)
        if n == 1:
            ops.encode_attention_q4(d_q, d_k, d_v, d_out, scratch, row + 1, max_seq, heads, n_kv, hd, weights=d_w)
        else:
            ops.encode_attention_prefill_q4(d_q, heads * hd, d_k, d_v, d_out, heads * hd, scratch, row, n, max_seq, heads, n_kv, hd, weights=d_w)
        assert_f32_parity(d_out.download(np.float32, n * heads * hd).reshape(n, heads, hd), ref, f"{n} tokens at row {row}")
        w[:, :row + n] += R.gathered(p, n_kv)
        got_w = back(d_w, w)
        assert_f32_parity(got_w, w, f"weights behind {n} tokens at row {row}")
        w, pos, row = got_w, pos + n, row + n
    assert pos > max_seq - 20 and row < max_seq


# ---- operands of unlike sizes -----------------------------------------------------------------------
# An operand is held as two halves of a row that is scaled by a power of two so that its largest value is below 2^15 (a softmax weight: the largest is
# 2^15): of a value x, 22 bits are left, or what is above 2^-25 of the scaled row, so it is off by at most max(2^-22 |x|, 2^-40 of the row's largest).

def run_attention(ctx, ops, dev, q, k, v, pos0, weights=True):
    """(out, weights gathered from zero) of n tokens at pos0 .., by the form for one token where it is one."""
    n, heads, hd = q.shape
    n_kv, max_seq = k.n_kv, k.max_seq
    scratch, d_out = scratch_for(ctx, dev, n, max_seq, heads, n_kv, hd, weights), dev(np.full(q.shape, np.nan, np.float32))
    d_w = dev(np.zeros((n_kv, max_seq), np.float32)) if weights else None
    if n == 1:
        ops.encode_attention_q4(dev(q), dev(k.raw), dev(v.raw), d_out, scratch, pos0 + 1, max_seq, heads, n_kv, hd, weights=d_w)
    else:
        ops.encode_attention_prefill_q4(dev(q), heads * hd, dev(k.raw), dev(v.raw), d_out, heads * hd, scratch, pos0, n, max_seq, heads, n_kv, hd, weights=d_w)
    return back(d_out, q), d_w.download(np.float32, n_kv * max_seq).reshape(n_kv, max_seq) if weights else None


EITHER_KERNEL = [  # head_dim, heads, KV heads, first row, tokens: a token, a few, more than 12 million pairs
    (64, 4, 2, 1500, 1), (128, 8, 2, 700, 20), (32, 4, 1, 900, 30), (256, 4, 2, 500, 1),
    (64, 16, 4, 1200, 700), (128, 16, 4, 1000, 700), (32, 16, 2, 1000, 1000), (256, 8, 2, 1700, 800),
]


@pytest.mark.parametrize("r", [10, 100, 1000, 10000])
@pytest.mark.parametrize("hd,heads,n_kv,pos0,n", EITHER_KERNEL)
def test_large_key_channels_meet_small_query_channels(ctx, ops, dev, hd, heads, n_kv, pos0, n, r):
    """Some channels of the keys r times as large as the others and those of the queries r times as small: all of them have their part in a score.  A score
    q.k / sqrt(hd) of normal values has addends that sum up to about 0.64 sqrt(hd) in magnitude (13 at most: heads of 256, queries of twice the spread: 26), each off by
    2^-22: 6e-6 if all were off the same way, a tenth of that as they are not; the bar of f32 outputs is 1e-5.  (An absolute 2^-25 of a row's largest: 9e-5 at r = 1000.)"""
    seq = pos0 + n
    size = np.ones(hd, np.float32)
    size[:16 if hd == 32 else 32] = r
    k, v = R.Cache(seq, n_kv, hd), R.Cache(seq, n_kv, hd)
    k.append(0, normal(r, seq, n_kv, hd) * size), v.append(0, normal(r + 1, seq, n_kv, hd))
    assert np.isfinite(k.scales).all()
    q = normal(r + 2, n, heads, hd) / size
    ref, p = R.attention(q, k, v, pos0)
    out, w = run_attention(ctx, ops, dev, q, k, v, pos0)
    assert_f32_parity(out, ref, "out")
    assert_f32_parity(w, R.gathered(p, n_kv), "weights")


@pytest.mark.parametrize("hd,heads,n_kv,pos0,n", [(64, 16, 4, 31, 1), (64, 16, 2, 1999, 1), (32, 16, 1, 31, 1), (128, 16, 4, 31, 1), (256, 16, 2, 31, 1), (128, 16, 4, 20, 12),
                                                  (64, 16, 4, 700, 900), (128, 16, 4, 700, 900), (32, 16, 4, 500, 1200), (256, 16, 2, 700, 900)])
def test_a_first_row_that_draws_nearly_all_weight(ctx, ops, dev, hd, heads, n_kv, pos0, n):
    """Its value is zero, the others' are one and their weights alike, so that their roundings add up.  Each is off by at most 2^-22 of itself or 2^-40 of the largest
    (relative to the largest: 2^-40).  Besides, the first row's score, `lead`, is off by what f32 leaves of it, and an output by as much, relative: the queries'
    halves 2^-22; its factor and their product 3 roundings of 2^-24; its sum, of addends of one sign, hd / 16 steps of three matrix instructions that each round, or cut
    off, the sum so far at 2^-23 (half of the whole on average).  1e-6 for the exponentials, sums and the division (some 2^-23 each)."""
    seq = pos0 + n
    k, v = R.Cache(seq, n_kv, hd), R.Cache(seq, n_kv, hd)
    x = np.zeros((seq, n_kv, hd), np.float32)
    x[0] = 1.0
    k.append(0, x), v.append(0, 1.0 - x)
    lead = np.linspace(10.0, 20.0, heads) + 0.37 * np.arange(n)[:, None] / n  # of the first row's score, by head and token
    q = np.broadcast_to((lead / np.sqrt(hd))[..., None], (n, heads, hd)).astype(np.float32)
    ref, _ = R.attention(q, k, v, pos0)
    out, _ = run_attention(ctx, ops, dev, np.ascontiguousarray(q), k, v, pos0, weights=False)
    rows = np.arange(pos0, seq)[:, None, None]  # of the others, by token
    of_a_score = 2.0 ** -22 + 3 * 2.0 ** -24 + 3 * hd / 16 / 2 * 2.0 ** -23
    off = np.abs(out - ref) / ((lead[..., None] * of_a_score + 1e-6) * np.abs(ref) + 2.0 ** -40 * rows)
    assert off.max() <= 1, f"{off.max():.2f} of what it may be off by, head and token {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("unit", [2.0 ** -149, 2.0 ** -148, 2.0 ** -140, 2.0 ** -126, 2.0 ** -101])
@pytest.mark.parametrize("hd,heads,n_kv,pos0,n", EITHER_KERNEL)
def test_queries_of_the_smallest_floats(ctx, ops, dev, hd, heads, n_kv, pos0, n, unit):
    """Rows whose largest value is one to three units: every score rounds to nothing, all rows that a token sees weigh alike."""
    seq = pos0 + n
    k, v = filled(n, seq, n_kv, hd, seq)
    q = (np.random.default_rng(1).integers(-3, 4, (n, heads, hd)) * unit).astype(np.float32)
    q[:, 0] = np.clip(q[:, 0], -unit, unit)
    assert np.all((q[:, 0] != 0).any(-1)) and np.abs(q[:, 0]).max() == unit
    ref, p = R.attention(q, k, v, pos0)
    out, w = run_attention(ctx, ops, dev, q, k, v, pos0)
    assert_f32_parity(out, ref, "out")
    assert_f32_parity(w, R.gathered(p, n_kv), "weights")


# ---- weights from zero, and many splits -------------------------------------------------------------

@pytest.mark.parametrize("hd,heads,n_kv,seq,max_seq", DECODE + [(64, 4, 1, 20000, 20100), (128, 8, 2, 30000, 30000), (256, 4, 1, 15000, 15000), (32, 8, 4, 12289, 13000)])
def test_weights_of_one_token_from_zero(ctx, ops, dev, hd, heads, n_kv, seq, max_seq):
    """Held to the bar by themselves, not as what they change in a sum.  The last four: more than 64 splits in use (128 rows each at the least), each by value and
    from device memory."""
    k, v = filled(seq, max_seq, n_kv, hd, seq)
    q = 2 * normal(seq + 5, 1, heads, hd)
    out, p = R.attention(q, k, v, seq - 1)
    scratch, d_k, d_v, d_q = scratch_for(ctx, dev, 1, max_seq, heads, n_kv, hd, True), dev(k.raw), dev(v.raw), dev(q)
    for d_pos in (None, dev(np.array([seq - 1], np.uint32))):
        d_out, d_w = dev(np.full(heads * hd, np.nan, np.float32)), dev(np.zeros((n_kv, max_seq), np.float32))
        ops.encode_attention_q4(d_q, d_k, d_v, d_out, scratch, seq if d_pos is None else 0, max_seq, heads, n_kv, hd, weights=d_w, d_pos=d_pos)
        assert_f32_parity(d_out.download(np.float32, heads * hd).reshape(heads, hd), out[0], f"d_pos {d_pos}")
        got = d_w.download(np.float32, n_kv * max_seq).reshape(n_kv, max_seq)
        assert_f32_parity(got[:, :seq], R.gathered(p, n_kv), "weights")
        assert not got[:, seq:].any()


@pytest.mark.parametrize("hd,heads,n_kv,pos0,n", [(64, 5, 5, 40000, 3), (64, 2, 1, 30000, 40)] + [p[:5] for p in LARGE])
def test_weights_of_a_prompt_from_zero(ctx, ops, dev, hd, heads, n_kv, pos0, n):
    k, v = filled(n, pos0 + n, n_kv, hd, pos0 + n)
    q = 2 * normal(n + 5, n, heads, hd)
    p = R.attention(q, k, v, pos0)[1]
    assert_f32_parity(run_attention(ctx, ops, dev, q, k, v, pos0)[1], R.gathered(p, n_kv), "weights")
