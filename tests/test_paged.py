"""Calls on KV caches in pages and of sampling without a GPU: the refusals of the library's host code against a pretended HIP runtime, and the numpy forms that
the GPU tests compare with."""
import numpy as np
import pytest

import paged_ref as R
from test_kv_q4 import run_host


def test_calls_that_are_refused(tmp_path):
    run_host("paged_calls", tmp_path)


def whole(pool):
    """What a pool says of itself fits together."""
    for s, (held, n) in enumerate(zip(pool.held, pool.lens)):
        assert len(held) == -(-n // pool.R) and len(set(held)) == len(held), s
        assert np.array_equal(pool.table[s, :len(held)], held) and np.all(pool.table[s, len(held):] == R.NONE)
    assert pool.refs.sum() == sum(map(len, pool.held))


@pytest.mark.parametrize("seed", range(6))
def test_lists_of_pages_through_a_life(seed):
    """Rows that a sequence has appended read back whatever others do: forks, cuts, moves, reservations that copy and those that do not fit."""
    rng = np.random.default_rng(seed)
    pool = R.Pool(5, 6, 14, 16, 1, 2, 0)
    rows, refused = [np.zeros((0, 2), np.float32) for _ in range(pool.S)], 0
    for step in range(120):
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            counts = [int(c) for c in rng.integers(0, 1 + int(rng.choice([1, 6, 40])), pool.S)]
            before = (pool.table.copy(), list(pool.lens))
            start, moves, wanting = pool.reserve(counts)
            refused += wanting != 0
            if wanting:
                assert np.array_equal(pool.table, before[0]) and pool.lens == before[1] and moves == [] and start == [R.NONE] * pool.S
                continue
            pool.copy(moves)
            refs = pool.refs
            for s, c in enumerate(counts):
                assert start[s] == (len(rows[s]) if c else R.NONE)
                x = rng.standard_normal((c, 2)).astype(np.float32)
                for i in range(c):
                    assert refs[pool.held[s][(start[s] + i) // pool.R]] == 1
                    pool.put(s, start[s] + i, x[i:i + 1], x[i:i + 1])
                rows[s] = np.concatenate([rows[s], x])
        elif what == "fork":
            parents = [s if rng.random() < 0.6 else int(rng.integers(0, pool.S + 1)) for s in range(pool.S)]
            pool.fork(parents)
            rows = [rows[p] if p < pool.S else rows[0][:0] for p in parents]
        elif what == "free":
            keep = [R.NONE if rng.random() < 0.6 else int(rng.integers(0, 60)) for _ in range(pool.S)]
            pool.free(keep)
            rows = [r[:k] for r, k in zip(rows, keep)]
        else:
            moves, used = pool.compact()
            pool.copy(moves)
            assert all(p < used for h in pool.held for p in h) and all(a >= used > b for a, b, _ in moves)
        whole(pool)
        for s in range(pool.S):
            assert pool.lens[s] == len(rows[s]) and np.array_equal(pool.rows(s, 1)[0].astype(np.float32), rows[s])
    assert refused


def test_attention_of_the_numpy_form():
    pool = R.Pool(3, 3, 7, 16, 2, 32, 0)
    pool.reserve([20, 0, 1])
    pool.planes[:] = np.random.default_rng(1).standard_normal(pool.planes.shape)
    q = np.random.default_rng(2).standard_normal((3, 4, 32)).astype(np.float32)
    out = pool.attention(q)
    assert np.all(out[1] == 0) and np.allclose(out[2], pool.rows(2, 1)[:, 0].repeat(2, 0))
    x = np.array([pool.rows(0, 0)[1, i] @ q[0, 3].astype(np.float64) for i in range(20)]) / np.sqrt(32)
    assert np.allclose(out[0, 3], np.exp(x) / np.exp(x).sum() @ pool.rows(0, 1)[1])
    seen = {0: np.arange(20) != 5}
    assert np.all(pool.attention(q, seen={0: np.zeros(20, bool)})[0] == 0) and not np.allclose(pool.attention(q, seen=seen)[0], out[0])


INF = np.inf


@pytest.mark.parametrize("logits,rule,tokens", [
    ([1, 3, 2, 3], (1.0, 1, 1.0, 0.0), [1]), ([1, 3, 2, 3], (1.0, 2, 1.0, 0.0), [1, 3]), ([1, 3, 2, 3], (0.0, 0, 1.0, 0.0), [1]), ([1, 3, 2, 3], (np.nan, 3, 0.5, 0.0), [1]),
    ([0, 0, 0, 0], (1.0, 0, 0.5, 0.0), [0, 1]), ([0, 0, 0, 0], (1.0, 0, 0.51, 0.0), [0, 1, 2]), ([0, 0, 0, 0], (1.0, 3, 0.5, 0.0), [0, 1]), ([0, 1], (1.0, 0, 0.0, 0.0), [1]),
    ([0, -1, -3], (1.0, 0, 1.0, 0.1), [0, 1]), ([0, -1, -3], (1.0, 0, 1.0, 5.0), [0]), ([0, 0, -3], (1.0, 0, 1.0, 5.0), [0, 1]), ([np.nan, -INF, 2], (1.0, 0, 1.0, 0.0), [2]),
    ([-INF, np.nan], (1.0, 0, 0.9, 0.1), []), ([INF, 1, INF], (1.0, 0, 1.0, 0.0), [0, 2]), ([2, 2, 1], (1.0, 9, np.nan, np.nan), [0, 1, 2]),
])
def test_what_the_rule_keeps(logits, rule, tokens):
    index, w = R.kept(logits, *rule)
    assert index[w > 0].tolist() == tokens
    for u in (0.0, 0.3, 0.999, 1.0, -1.0, 7.0, np.nan):
        token, prob, _ = R.sample(logits, *rule, u)
        assert token == R.NONE and prob == 0 if not tokens else token in tokens and 0 < prob <= 1
    if tokens:
        assert R.sample(logits, *rule, 0.0)[0] == tokens[0] and R.sample(logits, *rule, 1.0)[0] == tokens[-1]


def test_picks_are_as_often_as_their_weights():
    """Uniform numbers on a grid: a token is picked for its share of them, off by one at each end."""
    logits = np.random.default_rng(3).standard_normal(30).astype(np.float32)
    n = 4000
    picks = np.bincount([R.sample(logits, 0.7, 12, 0.9, 0.02, (i + 0.5) / n)[0] for i in range(n)], minlength=30)
    index, w = R.kept(logits, 0.7, 12, 0.9, 0.02)
    want = np.zeros(30)
    want[index] = w / w.sum() * n
    assert np.all(np.abs(picks - want) <= 1) and (picks > 0).sum() == index.size < 12


@pytest.mark.parametrize("n", [30, 512, 1000])
def test_top_p_is_of_all_that_top_k_leaves(n):
    """Tokens that min-p rules out afterwards are part of the mass that top-p takes its share of."""
    for live, rule, tokens in (([1, 0.06, 0.055] + [0.01] * 27, (1.0, 40, 0.9, 0.05), 3), ([1, 0.9] + [0.1] * 20, (1.0, 40, 0.5, 0.3), 2)):
        logits = np.full(n, -INF, np.float32)
        logits[:len(live)] = np.log(live)
        index, w = R.kept(logits, *rule)
        assert index.tolist() == list(range(tokens)) and np.allclose(w, live[:tokens], rtol=1e-6)
        assert np.isclose(R.sample(logits, *rule, 0.0)[1], 1 / sum(live[:tokens]), rtol=1e-6)
