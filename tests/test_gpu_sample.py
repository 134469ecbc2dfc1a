"""Sampling on the GPU against the rule in f64 (paged_ref.py).  A pick may differ where the uniform number lies within 1e-9 of a border of the mass: masses are
whole numbers of 2^-43 of the largest token's, up to 2^19 of them each off by half of one."""
# (That is n 2^-44 of the largest weight for n tokens, at most 2^-25: 1e-9 of the mass bounds up to 17000 tokens whatever their weights.  The longer rows here stay below it because
# their masses are many times the largest weight, and because rounded weights are off to either side.)
import numpy as np
import pytest

import paged_ref as R
import wick_amd as W
from wick_amd import lfm2
from wick_amd.lfm2 import NO_TOKEN, Lfm2Ops

pytestmark = pytest.mark.gpu


@pytest.fixture()
def run(ctx):
    """(logits, [(temperature, top_k, top_p, min_p)], u) -> (tokens, probabilities)"""
    ops = Lfm2Ops(ctx)

    def go(logits, params, u, stride=None, prob=True):
        rows, n = logits.shape
        stride = stride or n
        wide = np.full((rows, stride), 1e9, np.float32)  # (what is behind a row would be taken)
        wide[:, :n] = logits
        bufs = [ctx.to_device(x) for x in (wide, lfm2.sample_params(params).view(np.uint32), np.asarray(u, np.float32), np.full(rows, 12345, np.uint32),
                                           np.full(rows, 2.0, np.float32), np.full(lfm2.sample_scratch_bytes(rows, n), 0xff, np.uint8))]
        ops.sample(bufs[0], stride, rows, n, bufs[1], bufs[2], bufs[3], bufs[4] if prob else None, bufs[5])
        got = bufs[3].download(np.uint32, rows), bufs[4].download(np.float32, rows)
        for b in bufs:
            b.free()
        return got

    return go


def check(got, logits, params, u):
    held = lfm2.sample_params(params).tolist()  # (as the call has them: f32)
    for r in range(len(logits)):
        token, prob, border = R.sample(logits[r], *held[r], u[r])
        if border < 1e-9:
            continue
        assert got[0][r] == token, (r, params[r], u[r], border)
        assert abs(got[1][r] - prob) <= 2.0 ** -24 * prob + 1e-9 * prob, (r, params[r])  # rounded once


def logits_of(seed, rows, n, spread=3.0):
    return (spread * np.random.default_rng(seed).standard_normal((rows, n))).astype(np.float32)


RULES = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.05), (0.3, 0, 0.9, 0.0), (1.6, 0, 0.99, 0.0), (1.0, 1, 1.0, 0.0), (0.0, 50, 0.5, 0.1), (-1.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.1),
         (0.7, 500, 1.0, 0.0), (1.2, 7, 0.6, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1e-6, 0.0), (2.0, 10 ** 9, 2.0, -1.0), (1.0, 0, 0.5, 1.0), (1.0, 0, 1.0, 7.0),
         (float("nan"), 5, 0.5, 0.0), (1.0, 20, float("nan"), float("nan")), (0.05, 100, 0.9, 0.01), (50.0, 0, 0.7, 0.0), (1.0, 2, 0.999, 0.5)]


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 4095, 4096, 4097, 8193, 50257, 65536])
def test_rules(run, n):
    """Every rule, at uniform numbers from one end to the other; rows with a stride of their own."""
    us = [0.0, 0.1, 0.37, 0.5, 0.93, 1 - 2.0 ** -24]
    params = [p for p in RULES for _ in us]
    u = np.array(us * len(RULES), np.float32)
    logits = logits_of(n, len(params), n)
    check(run(logits, params, u, stride=n + n % 5), logits, params, u)


def test_a_large_vocabulary(run):
    logits = logits_of(1, 6, 1 << 19)
    params, u = RULES[:6], np.linspace(0.05, 0.95, 6, dtype=np.float32)
    check(run(logits, params, u), logits, params, u)


def test_many_rows(run):
    logits = logits_of(2, 3000, 700)
    params, u = [RULES[r % len(RULES)] for r in range(3000)], np.random.default_rng(3).random(3000, dtype=np.float32)
    check(run(logits, params, u), logits, params, u)


@pytest.mark.parametrize("n", [5, 1024, 1025, 3000, 20000])
def test_equal_logits(run, n):
    """Ties go to the lowest index, whatever cuts them: all alike, two values, and whole numbers only."""
    rng = np.random.default_rng(n)
    logits = np.stack([np.zeros(n), np.full(n, -3.5), (np.arange(n) % 2) * 1.0, rng.integers(0, 4, n) * 1.0, rng.integers(-3, 1, n) * 0.5, -(np.arange(n) // 7 % 3) * 1.0]).astype(np.float32)
    logits = np.tile(logits, (len(RULES), 1))
    params, u = [p for p in RULES for _ in range(6)], np.random.default_rng(1).random(6 * len(RULES), dtype=np.float32)
    check(run(logits, params, u), logits, params, u)


def test_flat_rows_list_more_than_a_workgroup(run):
    """Logits so close together that the cut's bin holds thousands, none of them alike."""
    logits = logits_of(4, 8, 30000, spread=0.01)
    params, u = [(1.0, 777, 1.0, 0.0), (1.0, 20000, 0.5, 0.0), (1.0, 0, 0.3, 0.0), (1.0, 0, 0.999, 0.0), (1.0, 29999, 1.0, 0.0), (0.5, 1, 1.0, 0.0), (1.0, 15000, 0.9, 0.98),
                 (1.0, 12345, 0.00001, 0.0)], np.linspace(0.01, 0.99, 8, dtype=np.float32)
    check(run(logits, params, u), logits, params, u)


@pytest.mark.parametrize("min_p", [2.0 ** -149, 1e-13, 2.0 ** -43, 1e-6, 0.01, 0.25, 0.5, float(np.nextafter(np.float32(0.5), np.float32(1))), 0.999, 1.0])
def test_the_floor_alone(run, min_p):
    """Tokens on the floor and a step off it, on both sides; rows of infinities and of values whose 4 y leave what is exact."""
    n = 9000
    logits = logits_of(15, 6, n)
    logits[1] = (np.log(min_p) + 3 + np.arange(-4500, 4500) * 2.0 ** -20).astype(np.float32)
    logits[1, 4321] = 3.0
    logits[2] = np.log(2.0) * -(np.arange(n) % 60)
    logits[3] *= 1e18
    logits[4, :4000] = np.inf
    logits[5, 7:] = -np.inf
    u = np.array([0.7, 0.9, 0.5, 0.3, 0.6, 0.2], np.float32)
    params = [(1.0, 0, 1.0, min_p)] * 6
    check(run(logits, params, u), logits, params, u)


def test_long_lists(run):
    """Many times what a workgroup holds at once is listed: alike, two values, nearly alike, alike but for a few, and alike from somewhere on."""
    n, rng = 150001, np.random.default_rng(6)
    logits = np.stack([np.full(n, 2.5), np.where(np.arange(n) % 3 == 0, 1.0, 0.9), rng.standard_normal(n) * 1e-6, np.where(rng.random(n) > 1 - 1e-4, 1.0, 0.0),
                       np.where(np.arange(n) > 100000, 0.0, -1e-3 * rng.random(n))]).astype(np.float32)
    params = [(1.0, 100000, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (1.0, 40, 0.95, 0.05), (0.7, 140000, 0.8, 0.9)]
    logits, params = np.tile(logits, (len(params), 1)), [p for p in params for _ in range(5)]
    u = rng.random(len(params)).astype(np.float32)
    check(run(logits, params, u), logits, params, u)


def test_ruled_out_tokens(run):
    """-infinity and NaN are never taken; a row of nothing else has no token; one alone is taken for certain; the lowest float is a token like others."""
    n = 5000
    logits = logits_of(5, 8, n)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2], logits[2, 4321] = -np.inf, -7.0
    logits[3, ::2], logits[3, 1::4] = -np.inf, np.nan
    logits[4] = np.finfo(np.float32).min
    logits[5], logits[5, 17] = np.finfo(np.float32).min, 0.0
    logits[6, :4990] = np.nan
    logits[7] = np.where(np.arange(n) % 2, -np.inf, np.nan)
    for rule in RULES:
        params, u = [rule] * 8, np.array([0.5, 0.5, 0.999, 0.3, 0.25, 0.99, 0.6, 0.1], np.float32)
        got = run(logits, params, u)
        check(got, logits, params, u)
        assert got[0][0] == got[0][1] == got[0][7] == NO_TOKEN and got[1][0] == got[1][1] == got[1][7] == 0
        assert got[0][2] == 4321 and got[1][2] == 1 and got[0][3] % 4 == 3


def test_infinite_logits(run):
    """+infinity leaves nothing for the finite ones; several share alike."""
    logits = logits_of(6, 4, 900)
    logits[0, 700] = logits[1, 5] = logits[1, 800] = np.inf
    logits[2, :300], logits[2, 400] = np.inf, -np.inf
    logits[3] = np.inf
    u = np.array([0.9, 0.6, 0.5, 0.25], np.float32)
    for rule in [(1.0, 0, 1.0, 0.0), (0.7, 100, 0.9, 0.0), (1e-30, 0, 1.0, 0.5)]:
        got = run(logits, [rule] * 4, u)
        check(got, logits, [rule] * 4, u)
        assert got[0][0] == 700


@pytest.mark.parametrize("temperature", [1e-45, 1e-30, 1e-3, 1e6, 3e38, float("inf")])
def test_extreme_temperatures(run, temperature):
    logits = np.concatenate([logits_of(7, 2, 3000), logits_of(8, 1, 3000) * 1e30, logits_of(9, 1, 3000) * 1e-30])
    params, u = [(temperature, 0, 1.0, 0.0), (temperature, 10, 0.9, 0.0), (temperature, 0, 0.7, 0.0), (temperature, 0, 1.0, 0.1)], np.array([0.2, 0.7, 0.5, 0.4], np.float32)
    check(run(logits, params, u), logits, params, u)


def test_logits_far_from_zero(run):
    """A common offset takes no bits from what is between the logits."""
    base = np.round(logits_of(10, 4, 3000) * 16) / 16
    for offset in (-1e4, 300.0, 1e5):
        logits = (base + np.float32(offset)).astype(np.float32)
        params, u = RULES[:4], np.array([0.2, 0.7, 0.5, 0.4], np.float32)
        check(run(logits, params, u), logits, params, u)


def test_uniform_numbers_outside_their_range(run):
    logits = logits_of(11, 6, 300)
    u = np.array([-0.5, 1.0, 1.5, np.nan, np.inf, -np.inf], np.float32)
    got = run(logits, [(1.0, 0, 1.0, 0.0)] * 6, u)
    for r, last in enumerate((False, True, True, False, True, False)):
        assert got[0][r] == (299 if last else 0)


def test_without_probabilities_and_in_every_run_the_same(run):
    logits = logits_of(12, 50, 50257)
    params, u = [RULES[r % 4] for r in range(50)], np.random.default_rng(4).random(50, dtype=np.float32)
    a, b, c = run(logits, params, u), run(logits, params, u), run(logits, params, u, prob=False)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1]) and np.array_equal(a[0], c[0]) and np.all(c[1] == 2.0)


def test_picks_follow_the_probabilities(run):
    """Over a grid of uniform numbers every token comes up in proportion: the k-th of m equal steps is the f64 rule's."""
    m = 4000
    logits = np.repeat(logits_of(13, 1, 37), m, 0)
    u = ((np.arange(m) + 0.5) / m).astype(np.float32)
    got = run(logits, [(1.0, 20, 0.9, 0.01)] * m, u)
    index, w = R.kept(logits[0], 1.0, 20, 0.9, 0.01)
    assert np.all(np.diff(got[0].astype(int)) >= 0)
    share = np.bincount(got[0], minlength=37)[index] / m
    assert np.all(np.abs(share - w / w.sum()) <= 1.5 / m) and set(got[0]) <= set(index)


def test_greedy_rows_are_the_largest(ctx, run):
    """Where the largest logit is one alone, temperature 0 is wick_rocm_argmax."""
    logits = logits_of(14, 5, 65536)
    got = run(logits, [(0.0, 0, 1.0, 0.0)] * 5, np.zeros(5))
    out = ctx.alloc(4)
    for r in range(5):
        x = ctx.to_device(logits[r])
        Lfm2Ops(ctx).argmax(x, 65536, out)
        assert got[0][r] == out.download(np.uint32, 1)[0] and got[1][r] == 1
        x.free()
    out.free()


# (temperature, top_k, top_p, min_p) where the nucleus and min-p both cut, under a top_k that leaves at most 512 tokens
NUCLEUS_AND_FLOOR = [(0.8, 40, 0.95, 0.05), (1.0, 40, 0.5, 0.3), (1.0, 500, 0.9, 0.1), (0.1, 40, 0.9, 0.01), (1.0, 512, 0.8, 0.999)]


@pytest.mark.parametrize("n", [40, 512, 513, 5000, 20000])
def test_fewer_live_tokens_than_top_k(run, n):
    """Rows of which a grammar leaves fewer tokens than top_k: top-p's share is of all of them, min-p cuts what top-p leaves.  (At most 300 masses, each off by half of
    2^-43 where the largest is at least 1: within 2e-11 of the whole.)"""
    rng = np.random.default_rng(n)
    rules = NUCLEUS_AND_FLOOR + ([(1.0, 0, 0.7, 0.2)] if n <= 512 else [])
    us, logits, params = [0.05, 0.4, 0.75, 0.97], [], []
    for live in (2, 3, 5, 8, 13, 21, 30, 39, 64, 65, 120, 300):
        for rule in rules if live < n else []:
            for spread in (1.0, 2.5):
                row = np.full(n, -np.inf, np.float32)
                row[rng.permutation(n)[:live]] = spread * rng.standard_normal(live)
                logits += [row] * len(us)
                params += [rule] * len(us)
    u = np.array(us * (len(params) // len(us)), np.float32)
    logits = np.stack(logits)
    check(run(logits, params, u), logits, params, u)


@pytest.mark.parametrize("n", [30, 512, 1000, 70000])
def test_a_tail_below_the_floor_counts_for_the_nucleus(run, n):
    """Light tokens that min-p rules out are part of the mass that top-p takes its share of."""
    tail_of_27 = np.log(np.array([1, 0.06, 0.055] + [0.01] * 27))
    two_and_20 = np.log(np.array([1, 0.9] + [0.1] * 20))
    us = (np.arange(32, dtype=np.float32) + 0.5) / 32
    for live, rule, kept in ((tail_of_27, (1.0, 40, 0.9, 0.05), [1, 0.06, 0.055]), (two_and_20, (1.0, 40, 0.5, 0.3), [1, 0.9])):
        logits = np.full((32, n), -np.inf, np.float32)
        at = np.random.default_rng(n).permutation(n)[:live.size]
        logits[:, at] = live
        got = run(logits, [rule] * 32, us)
        assert set(got[0]) <= set(at[:len(kept)])
        check(got, logits, [rule] * 32, us)
        for token, w in zip(at, kept):  # (logits are f32: weights within 2^-23 or so)
            assert np.all(np.abs(got[1][got[0] == token] - w / sum(kept)) <= 1e-6)
        assert len(set(got[0])) == len(kept)


@pytest.mark.parametrize("temperature", [0.02, 0.1])
def test_cold_rows_of_a_whole_vocabulary(run, temperature):
    """At low temperatures few of many finite tokens have mass."""
    logits = logits_of(16, 120, 50257, spread=4.0)
    params, u = [(temperature, 40, 0.9, 0.05), (temperature, 200, 0.6, 0.02), (temperature, 512, 0.99, 0.1)] * 40, np.random.default_rng(17).random(120, dtype=np.float32)
    check(run(logits, params, u), logits, params, u)
