"""The operators around a KV cache held in 4 bits, as cases that can be timed: rows appended to it and read back, attention of a single
token and of a prompt over it (with the attention weight that its rows have gathered, where a case asks for it), and the eviction of the
rows that gathered least.  `own` chooses between their plain form in torch and the framework's entry points."""
import math

import numpy as np
import torch

own = False

# A cache, as the framework documents it: for every KV head and row 32-element blocks of 4-bit values, 8 consecutive values to a
# 32-bit word (value 2 i in bits 4 i .., value 2 i + 1 in bits 16 + 4 i ..), behind all of them one f16 scale per block; a value stands
# for (nibble - 8) * scale.
SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]
LARGEST = 65504.0  # of a value that a cache can hold


def listed():
    return [
        # a decode step's new key and value heads, the smaller model's: all launch and latency
        {"name": "append_1", "kind": "append", "n": 1, "row": 700, "kv": 8, "hd": 64},
        # a pass of a long prompt
        {"name": "append_2002", "kind": "append", "n": 2002, "row": 0, "kv": 8, "hd": 64},
        # a step right behind a short prompt
        {"name": "step_pos30", "kind": "step", "pos": 30, "heads": 16, "kv": 8, "hd": 64, "weights": False},
        # a step in the middle of a chat that evicts rows: the weights are gathered
        {"name": "step_pos9000_weights", "kind": "step", "pos": 9000, "heads": 16, "kv": 8, "hd": 64, "weights": True},
        # a step far into a long context, the larger model's heads
        {"name": "step_pos20000", "kind": "step", "pos": 20000, "heads": 32, "kv": 8, "hd": 64, "weights": False},
        # a step at the end of the longest context, wide heads: all reading
        {"name": "step_pos127999_hd128", "kind": "step", "pos": 127999, "heads": 32, "kv": 8, "hd": 128, "weights": False},
        # a chat turn: a few tokens onto an existing context
        {"name": "prompt_23_at700", "kind": "prompt", "n": 23, "pos": 700, "heads": 16, "kv": 8, "hd": 64, "weights": False},
        # an ordinary prompt whose weights are gathered
        {"name": "prompt_555_weights", "kind": "prompt", "n": 555, "pos": 0, "heads": 16, "kv": 8, "hd": 64, "weights": True},
        # a long prompt, the larger model's heads
        {"name": "prompt_2002", "kind": "prompt", "n": 2002, "pos": 0, "heads": 32, "kv": 8, "hd": 64, "weights": False},
        # a pass of a document, behind three others, wide heads
        {"name": "prompt_2048_at6144_hd128", "kind": "prompt", "n": 2048, "pos": 6144, "heads": 16, "kv": 4, "hd": 128, "weights": False},
        # a chat makes room
        {"name": "evict_800_of_3000", "kind": "evict", "seq": 3000, "keep": 64, "recent": 256, "drop": 800, "kv": 8, "hd": 64},
        # a document's cache cut to three quarters
        {"name": "evict_8192_of_32768", "kind": "evict", "seq": 32768, "keep": 4, "recent": 1024, "drop": 8192, "kv": 8, "hd": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "step", "step", "prompt", "prompt", "evict"])
    hd, kv = rng.choice([32, 64, 64, 128, 256]), rng.choice([1, 2, 3, 4, 8])
    c = {"kind": kind, "kv": kv, "hd": hd}
    if kind == "append":
        c.update(n=_log(rng, 1, 4096), row=_log(rng, 1, 8000))
    elif kind == "evict":
        seq = _log(rng, 64, 32768)
        drop = rng.randint(1, seq // 2)
        keep = rng.randint(0, min(64, seq - drop))
        c.update(seq=seq, keep=keep, recent=rng.randint(0, seq - drop - keep), drop=drop)
    else:
        c.update(heads=kv * rng.choice([1, 2, 3, 4, 8]), weights=rng.random() < 0.4)
        if kind == "step":
            c.update(pos=min(_log(rng, 1, 120000), 120000 * 8 * 128 // (kv * hd)))
        else:
            n = _log(rng, 2, 2048)
            pos = 0 if rng.random() < 0.4 else _log(rng, 16, 6000)
            most = 4e10 / (c["heads"] * hd)  # pairs of a token and a row
            n = max(2, min(n, int(math.sqrt(pos * pos + 2 * most) - pos)))
            c.update(n=n, pos=pos)
    return c


# ---- inputs ----------------------------------------------------------------------------------

def _quantize(x):
    """(nibbles, f16 scales) of [..., 32 k] floats in blocks of 32.  The rule is stated in 32-bit steps, so that every nibble is decided:
    each product, quotient and sum is taken in 64 bits, where it is exact or as good as, and rounded to 32 once."""
    b = x.unflatten(-1, (-1, 32))
    high, low = b.amax(-1, keepdim=True), b.amin(-1, keepdim=True)
    d = torch.where(high >= -low, high, low) / -8.0  # the value of largest magnitude, the positive one of two
    held = torch.where(b.abs().amax(-1, keepdim=True) <= LARGEST, d, math.nan).half()  # (false for NaN too)
    full = held.abs() > 0  # a block without a scale holds nothing: zeros, or NaN
    inverse = (1.0 / torch.where(full, d, 1.0).double()).float()
    t = torch.where(full, (b.double() * inverse.double()).float(), 0.0)
    nibble = (t.double() + 8.5).float().clamp(max=15.0).to(torch.uint8)
    return nibble.flatten(-2), held.squeeze(-1)


def _shift(device):
    return torch.tensor(SHIFTS, device=device, dtype=torch.int64)


def _planes(cache, c):
    """A cache's words [kv][rows][hd / 8] and scales [kv][rows][hd / 32], as views."""
    rows, kv, hd = _rows(c), c["kv"], c["hd"]
    quants = kv * rows * hd // 2
    return cache[:quants].view(torch.int32).view(kv, rows, hd // 8), cache[quants:].view(torch.float16).view(kv, rows, hd // 32)


def _store(cache, c, row, x):
    """Rows [row, row + n) of a cache from [n][kv][hd] floats."""
    n = x.shape[0]
    words, scales = _planes(cache, c)
    nibble, d = _quantize(x.transpose(0, 1))
    w = (nibble.unflatten(-1, (-1, 8)).long() << _shift(x.device)).sum(-1)
    words[:, row:row + n] = torch.where(w >= 1 << 31, w - (1 << 32), w).int()
    scales[:, row:row + n] = d


def _values(cache, c, row, n):
    """Rows [row, row + n) of a cache as [kv][n][hd] floats."""
    words, scales = _planes(cache, c)
    nibble = (words[:, row:row + n].long().unsqueeze(-1) >> _shift(cache.device)) & 15
    v = (nibble.flatten(-2).unflatten(-1, (-1, 32)) - 8).float() * scales[:, row:row + n].float().unsqueeze(-1)
    return v.flatten(-2)


def _rows(c):
    """Rows of the case's caches: some more than are in use, as a program has them."""
    used = {"append": lambda: c["row"] + c["n"], "step": lambda: c["pos"] + 1, "prompt": lambda: c["pos"] + c["n"], "evict": lambda: c["seq"]}[c["kind"]]()
    return (used + 255) // 256 * 256


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    c, kind = dict(case), case["kind"]
    kv, hd, rows = c["kv"], c["hd"], _rows(c)
    size = kv * rows * (hd // 2 + hd // 16)
    st = {"case": c, "rows": rows, "k_cache": torch.zeros(size, dtype=torch.uint8, device="cuda"), "v_cache": torch.zeros(size, dtype=torch.uint8, device="cuda")}
    if kind == "append":
        # normed and rotated keys of unit spread, values of a spread of their own for each head
        st["k"], st["v"] = normal(c["n"], kv * hd), (normal(c["n"], kv, hd) * torch.exp(normal(kv, 1))).flatten(1)
        st["k_back"], st["v_back"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    else:
        used = {"step": c.get("pos", 0) + 1, "prompt": c.get("pos", 0) + c.get("n", 0), "evict": c.get("seq")}[kind]
        channel = torch.exp(0.3 * normal(kv, hd))  # some channels of the keys are larger than others
        _store(st["k_cache"], c, 0, normal(used, kv, hd) * channel)
        _store(st["v_cache"], c, 0, normal(used, kv, hd))
    if kind in ("step", "prompt"):
        n, heads = c.get("n", 1), c["heads"]
        st["q"], st["out"] = 1.5 * normal(n, heads * hd), torch.empty(n, heads * hd, device="cuda")
        if c["weights"]:
            st["weights"] = torch.exp(2.0 * normal(kv, rows)) * 0.01
    if kind == "evict":
        # a few rows gather most of the weight, some none at all
        st["weights"] = torch.exp(2.0 * normal(kv, rows)) * (torch.rand(kv, rows, generator=gen, device="cuda") > 0.05)
        st["kept"] = torch.zeros(kv, c["seq"] - c["drop"], dtype=torch.int32, device="cuda")
        st["k_back"], st["v_back"] = (torch.empty(c["seq"] - c["drop"], kv * hd, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    return st


# ---- the operators in their plain form -----------------------------------------------------------

def _attend(st):
    c = st["case"]
    n, pos, kv, hd = c.get("n", 1), c["pos"], c["kv"], c["hd"]
    group = c["heads"] // kv
    k, v = _values(st["k_cache"], c, 0, pos + n), _values(st["v_cache"], c, 0, pos + n)
    q = st["q"].view(n, kv, group, hd).permute(1, 2, 0, 3).reshape(kv, group * n, hd)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv, group, n, pos + n) / math.sqrt(hd)
    seen = torch.arange(pos + n, device="cuda") <= torch.arange(pos, pos + n, device="cuda").unsqueeze(1)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(kv, group * n, pos + n), v).view(kv, group, n, hd)
    st["out"].copy_(out.permute(2, 0, 1, 3).reshape(n, c["heads"] * hd))
    if c["weights"]:
        st["weights"][:, :pos + n] += p.sum((1, 2))


def _evict(st):
    c = st["case"]
    seq, left = c["seq"], c["seq"] - c["drop"]
    w = st["weights"]
    leave = torch.sort(w[:, c["keep"]:seq - c["recent"]], stable=True).indices[:, :c["drop"]] + c["keep"]  # (of equal ones the lower row first)
    stays = torch.ones(c["kv"], seq, dtype=torch.bool, device="cuda").scatter_(1, leave, False)
    kept = stays.nonzero()[:, 1].view(c["kv"], left)
    st["kept"].copy_(kept)
    for plane in (*_planes(st["k_cache"], c), *_planes(st["v_cache"], c)):
        plane[:, :left] = plane.gather(1, kept.unsqueeze(-1).expand(-1, -1, plane.shape[-1]))
    w[:, :left] = w.gather(1, kept)
    w[:, left:seq] = 0.0


def _read(cache, c, row, n, to):
    to.copy_(_values(cache, c, row, n).transpose(0, 1).flatten(1))


# ---- the framework's ---------------------------------------------------------------------------

_KEPT = {}  # what a program makes once: its context, and one workspace that all its calls share


def _ops():
    if not _KEPT:
        import wick_amd
        from wick_amd import lfm2

        ctx = wick_amd.RocmContext(0)
        _KEPT.update(lfm2=lfm2, ops=lfm2.Lfm2Ops(ctx), scratch=torch.empty(0, device="cuda"))
    return _KEPT["ops"]


def _workspace(floats):
    if _KEPT["scratch"].numel() < floats:
        torch.cuda.synchronize()
        _KEPT["scratch"] = torch.empty(floats, device="cuda")
    return _KEPT["scratch"].data_ptr()


def _run_own(st):
    c, kind, rows = st["case"], st["case"]["kind"], st["rows"]
    kv, hd, ops = c["kv"], c["hd"], _ops()
    k, v = st["k_cache"].data_ptr(), st["v_cache"].data_ptr()
    weights = st["weights"].data_ptr() if "weights" in st else None
    if kind == "append":
        ops.encode_kv_q4_append(st["k"].data_ptr(), st["v"].data_ptr(), kv * hd, k, v, c["row"], c["n"], rows, kv, hd)
        ops.encode_kv_q4_read(k, st["k_back"].data_ptr(), kv * hd, c["row"], c["n"], rows, kv, hd)
        ops.encode_kv_q4_read(v, st["v_back"].data_ptr(), kv * hd, c["row"], c["n"], rows, kv, hd)
    elif kind == "evict":
        left = c["seq"] - c["drop"]
        scratch = _workspace(_KEPT["lfm2"].kv_q4_evict_scratch_floats(c["seq"], kv))
        ops.encode_kv_q4_evict(k, v, weights, st["kept"].data_ptr(), scratch, c["seq"], c["keep"], c["recent"], c["drop"], rows, kv, hd)
        ops.encode_kv_q4_read(k, st["k_back"].data_ptr(), kv * hd, 0, left, rows, kv, hd)
        ops.encode_kv_q4_read(v, st["v_back"].data_ptr(), kv * hd, 0, left, rows, kv, hd)
    else:
        heads, n = c["heads"], c.get("n", 1)
        scratch = _workspace(_KEPT["lfm2"].attention_q4_scratch_floats(n, rows, heads, kv, hd, c["weights"]))
        q, out = st["q"].data_ptr(), st["out"].data_ptr()
        if kind == "step":
            ops.encode_attention_q4(q, k, v, out, scratch, c["pos"] + 1, rows, heads, kv, hd, weights=weights)
        else:
            ops.encode_attention_prefill_q4(q, heads * hd, k, v, out, heads * hd, scratch, c["pos"], n, rows, heads, kv, hd, weights=weights)


def _run_plain(st):
    c, kind = st["case"], st["case"]["kind"]
    if kind == "append":
        _store(st["k_cache"], c, c["row"], st["k"].view(c["n"], c["kv"], c["hd"]))
        _store(st["v_cache"], c, c["row"], st["v"].view(c["n"], c["kv"], c["hd"]))
        _read(st["k_cache"], c, c["row"], c["n"], st["k_back"])
        _read(st["v_cache"], c, c["row"], c["n"], st["v_back"])
    elif kind == "evict":
        _evict(st)
        _read(st["k_cache"], c, 0, c["seq"] - c["drop"], st["k_back"])
        _read(st["v_cache"], c, 0, c["seq"] - c["drop"], st["v_back"])
    else:
        _attend(st)


def run(st):
    if own:
        _run_own(st)
    else:
        _run_plain(st)
    names = {"append": ("k_back", "v_back"), "evict": ("kept", "weights", "k_back", "v_back")}.get(st["case"]["kind"], ("out", "weights"))
    return {name: st[name] for name in names if name in st}


# ---- what the outputs should be ----------------------------------------------------------------------

def _by_the_bits(cache, c, head, row, n):
    """Rows of one KV head from the cache's bytes, in 64 bits."""
    hd, rows = c["hd"], _rows(c)
    raw = cache[(head * rows + row) * hd // 2:(head * rows + row + n) * hd // 2].view(n, hd // 8, 4).int()
    out = torch.empty(n, hd // 8, 8, dtype=torch.float64, device=cache.device)
    for i, (byte, high) in enumerate(((0, 0), (2, 0), (0, 1), (2, 1), (1, 0), (3, 0), (1, 1), (3, 1))):
        out[..., i] = ((raw[..., byte] >> 4 * high) % 16).double() - 8
    at = c["kv"] * rows * hd // 2 + (head * rows + row) * hd // 16
    d = cache[at:at + n * hd // 16].view(torch.float16).double().view(n, hd // 32, 1)
    return (out.view(n, hd // 32, 32) * d).view(n, hd)


def exact(case, seed):
    st, c = prepare(case, seed), dict(case)
    kv, hd = c["kv"], c["hd"]
    if c["kind"] == "append":
        back = {}
        for name in ("k", "v"):
            # block by block by the rule's own steps (32-bit ones: numpy's are)
            x = st[name].cpu().numpy().reshape(-1, 32)
            m = x.max(1, keepdims=True)
            d = np.where(m >= -x.min(1, keepdims=True), m, x.min(1, keepdims=True)) / np.float32(-8)
            steps = (x * (np.float32(1) / d) + np.float32(8.5)).astype(np.int64).clip(max=15) - 8
            back[name + "_back"] = torch.from_numpy((steps * d.astype(np.float16).astype(np.float64)).reshape(c["n"], kv * hd))
        return back
    if c["kind"] == "evict":
        seq, left = c["seq"], c["seq"] - c["drop"]
        w = st["weights"].cpu().numpy()
        kept = np.empty((kv, left), np.int64)
        weights = w.astype(np.float64)
        back = {"k_back": torch.empty(left, kv, hd, dtype=torch.float64), "v_back": torch.empty(left, kv, hd, dtype=torch.float64)}
        for head in range(kv):
            rows = range(c["keep"], seq - c["recent"])
            gone = set(sorted(rows, key=lambda r: (w[head, r], r))[:c["drop"]])
            kept[head] = [r for r in range(seq) if r not in gone]
            weights[head, :left], weights[head, left:seq] = w[head, kept[head]], 0
            at = torch.from_numpy(kept[head]).cuda()
            for name in ("k", "v"):
                back[name + "_back"][:, head] = _by_the_bits(st[name + "_cache"], c, head, 0, seq)[at].cpu()
        return {"kept": None, "weights": torch.from_numpy(weights), "k_back": back["k_back"].flatten(1), "v_back": back["v_back"].flatten(1)}
    n, pos, heads = c.get("n", 1), c["pos"], c["heads"]
    out = torch.empty(n, heads, hd, dtype=torch.float64, device="cuda")
    weights = st["weights"].double() if c["weights"] else None
    ahead = torch.full((n, pos + n), -math.inf, dtype=torch.float64, device="cuda").triu(pos + 1)
    for h in range(heads):
        head = h // (heads // kv)
        q = st["q"][:, h * hd:(h + 1) * hd].double()
        p = torch.softmax(q @ _by_the_bits(st["k_cache"], c, head, 0, pos + n).T * hd ** -0.5 + ahead, -1)
        out[:, h] = p @ _by_the_bits(st["v_cache"], c, head, 0, pos + n)
        if weights is not None:
            weights[head, :pos + n] += p.sum(0)
    return {"out": out.flatten(1)} if weights is None else {"out": out.flatten(1), "weights": weights}


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    c = case
    kv, hd = c["kv"], c["hd"]
    row = kv * (hd // 2 + hd // 16)  # bytes of a row in one cache
    if c["kind"] == "append":  # (read back too)
        return {"bytes": c["n"] * (2 * row + 16 * kv * hd), "flops": 0}
    if c["kind"] == "evict":  # the dropped rows lie anywhere among those that may go: half of what is behind n_keep moves down at the least
        left = c["seq"] - c["drop"]
        return {"bytes": 8 * kv * c["seq"] + 4 * kv * left + 2 * row * (2 * (left - c["keep"])) + 8 * left * kv * hd, "flops": 0}
    n, pos, heads = c.get("n", 1), c["pos"], c["heads"]
    seen = n * pos + n * (n + 1) // 2
    w = {"bytes": 2 * (pos + n) * row + 8 * n * heads * hd, "flops": 4 * heads * hd * seen}
    if c["weights"]:
        w["bytes"] += 8 * kv * (pos + n)
    return w
