"""The operators around KV caches in pages that sequences share, as cases that can be timed: rows appended to pages, attention of one new
token of every sequence over them, what is done to pages themselves (a prompt's cache forked to several continuations, sequences that
come and go, the pool kept together), and the pick of the sequences' next tokens by temperature, top-k, top-p and min-p.  `own` chooses
between their plain form in torch and the framework's entry points."""
import math

import numpy as np
import torch

own = False

# A pool, as the framework documents it: planes (keys or values of a layer) of [n_pages][n_kv_heads][page_rows][head_dim]; table[s][i]
# names the page of rows [i page_rows, ..) of sequence s (-1: none), lens[s] its rows, refs[p] how many entries name page p.
TYPES = {"f32": torch.float32, "f16": torch.float16}
NONE = -1


def listed():
    return [
        # a decode step of one session in the middle of a chat: all launch and latency
        {"name": "attention_1_at700", "kind": "attention", "seqs": 1, "longest": 701, "heads": 16, "kv": 8, "hd": 64, "type": "f16", "rows": 16},
        # sessions of all lengths in one step, the larger model's heads
        {"name": "attention_32_ragged", "kind": "attention", "seqs": 32, "longest": 8192, "heads": 32, "kv": 8, "hd": 64, "type": "f16", "rows": 32},
        # many sessions over f32 rows (the CPU model's caches)
        {"name": "attention_64_f32", "kind": "attention", "seqs": 64, "longest": 2002, "heads": 32, "kv": 8, "hd": 64, "type": "f32", "rows": 64},
        # a step at the end of the longest context, wide heads: all reading
        {"name": "attention_1_at127999_hd128", "kind": "attention", "seqs": 1, "longest": 128000, "heads": 32, "kv": 8, "hd": 128, "type": "f16", "rows": 64},
        # a step's new rows, one a session
        {"name": "append_64", "kind": "append", "seqs": 64, "n": 64, "longest": 2002, "kv": 8, "hd": 64, "type": "f16", "rows": 32},
        # a prompt's rows, one session
        {"name": "append_2002", "kind": "append", "seqs": 1, "n": 2002, "longest": 2002, "kv": 8, "hd": 64, "type": "f32", "rows": 64},
        # a prompt continued 16 times: forked, the page that all would write to copied for each (six layers), the branches dropped again
        {"name": "branch_16_of_2002", "kind": "branch", "branches": 16, "length": 2002, "planes": 12, "kv": 8, "hd": 64, "type": "f16", "rows": 64},
        # the oldest of 32 sessions leaves, the pool is moved together, a new one is admitted (six layers)
        {"name": "turnover_32x2002", "kind": "turnover", "seqs": 32, "length": 2002, "planes": 12, "kv": 8, "hd": 64, "type": "f16", "rows": 64},
        # the same with long sessions in small pages
        {"name": "turnover_8x16000", "kind": "turnover", "seqs": 8, "length": 16000, "planes": 12, "kv": 8, "hd": 64, "type": "f16", "rows": 16},
        # a session's next token, the usual settings
        {"name": "sample_1x65536", "kind": "sample", "seqs": 1, "n": 65536, "mixed": False, "temperature": 0.8, "top_k": 40, "top_p": 0.95, "min_p": 0.05},
        # many continuations of one prompt: the nucleus of the whole vocabulary
        {"name": "sample_64x65536", "kind": "sample", "seqs": 64, "n": 65536, "mixed": False, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # sessions with settings of their own, an odd vocabulary
        {"name": "sample_200x50257_mixed", "kind": "sample", "seqs": 200, "n": 50257, "mixed": True, "temperature": 0.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "append", "branch", "turnover", "sample", "sample"])
    if kind == "sample":
        n = _log(rng, 1000, 200000)
        c = {"kind": kind, "seqs": min(_log(rng, 1, 256), max(1, 12000000 // n)), "n": n, "mixed": rng.random() < 0.3, "temperature": 0.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
        if not c["mixed"]:
            c.update(temperature=round(rng.uniform(0.3, 1.6), 3), top_k=rng.choice([0, 1, _log(rng, 2, 500)]), top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                     min_p=rng.choice([0.0, round(rng.uniform(0.005, 0.3), 3)]))
        return c
    c = {"kind": kind, "kv": rng.choice([1, 2, 3, 4, 8]), "hd": rng.choice([32, 64, 64, 128, 256]), "type": rng.choice(["f32", "f16", "f16"]), "rows": rng.choice([16, 32, 64, 128])}
    row = c["kv"] * c["hd"] * TYPES[c["type"]].itemsize  # bytes of a row in one plane
    if kind == "attention":
        seqs = _log(rng, 1, 100)
        c.update(seqs=seqs, heads=c["kv"] * rng.choice([1, 2, 3, 4, 8, 16]), longest=min(_log(rng, 1, 120000), max(1, 200000000 // (seqs * row))))
    elif kind == "append":
        seqs = _log(rng, 1, 64)
        c.update(seqs=seqs, n=_log(rng, seqs, 4096), longest=4096)
    else:
        c.update(planes=2 * rng.randint(1, 8), length=_log(rng, 20, 8000))
        most = max(3, 800000000 // (c["planes"] * row * (c["length"] + c["rows"])))
        c["branches" if kind == "branch" else "seqs"] = min(_log(rng, 2, 40), most)
    return c


# ---- inputs ----------------------------------------------------------------------------------

def _lengths(c):
    """Rows of the case's sequences: the longest first, the others spread over all lengths."""
    return [max(1, int(c["longest"] * (1.0 if i == 0 else i * 0.6180339887498949 % 1.0))) for i in range(c["seqs"])]


def _news(c):
    """Rows that a case's sequences get in one append."""
    return [c["n"] // c["seqs"] + (i < c["n"] % c["seqs"]) for i in range(c["seqs"])]


def _pages(n, c):
    return -(-n // c["rows"])


def _table(lens, max_pages, n_pages, c, gen):
    """A table whose sequences hold pages of their own, handed out as sequences grow side by side: no two neighbours together."""
    need = torch.tensor([_pages(n, c) for n in lens])
    table = torch.full((len(lens), max_pages), NONE, dtype=torch.int32)
    held = torch.arange(max_pages) < need.unsqueeze(1)
    ids = torch.randperm(int(need.sum()), generator=gen)
    table[held] = ids.int()
    refs = torch.zeros(n_pages, dtype=torch.int32)
    refs[ids] = 1
    return table, refs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    c, kind = dict(case), case["kind"]
    st = {"case": c}
    if kind == "sample":
        rows, n = c["seqs"], c["n"]
        # a few tokens stand out, some are ruled out (by a grammar, say)
        l = 2.5 * normal(rows, n) + 6.0 * (torch.rand(rows, n, generator=gen, device="cuda") > 1 - 20 / n) * torch.rand(rows, n, generator=gen, device="cuda")
        l[torch.rand(rows, n, generator=gen, device="cuda") > 0.98] = -math.inf
        st["logits"], st["u"] = l, torch.rand(rows, generator=gen, device="cuda")
        # temperature, top-k (whole), top-p, min-p of each row
        if c["mixed"]:
            r = torch.rand(rows, 6, generator=host)
            p = torch.stack([0.3 + 1.3 * r[:, 0], torch.where(r[:, 3] < 0.5, (1 + r[:, 1] * 200).floor(), 0.0), torch.where(r[:, 4] < 0.5, 0.5 + 0.49 * r[:, 2], 1.0),
                             torch.where(r[:, 5] < 0.3, 0.2 * r[:, 2], 0.0)], 1)
            p[r[:, 0] < 0.1, 0] = 0.0  # the largest
        else:
            p = torch.tensor([[c["temperature"], c["top_k"], c["top_p"], c["min_p"]]]).repeat(rows, 1)
        params = torch.empty(rows, 4, dtype=torch.int32)
        params[:, [0, 2, 3]], params[:, 1] = p[:, [0, 2, 3]].contiguous().view(torch.int32), p[:, 1].int()
        st["params"], st["token"], st["prob"] = params.cuda(), torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
        torch.cuda.synchronize()
        return st
    kv, hd, R, dtype = c["kv"], c["hd"], c["rows"], TYPES[c["type"]]
    if kind == "branch":
        lens, extra, moves = [c["length"]] + [0] * c["branches"], 2 * c["branches"] + 8, c["branches"] + 1
    elif kind == "turnover":
        lens = [c["length"]] * c["seqs"]
        extra = _pages(c["length"], c) + 8
    elif kind == "append":
        lens = [max(0, n - m) + m for n, m in zip(_lengths(c), _news(c))]
        extra = 4
    else:
        lens, extra = _lengths(c), 4
    max_pages = max(_pages(n, c) for n in lens) + 4
    n_pages = sum(_pages(n, c) for n in lens) + extra
    table, refs = _table(lens, max_pages, n_pages, c, host)
    st.update(n_pages=n_pages, max_pages=max_pages, table=table.cuda(), refs=refs.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda())
    shape = (n_pages, kv, R, hd)
    if kind in ("attention", "append"):
        channel = torch.exp(0.3 * normal(kv, 1, hd))  # some channels of the keys are larger than others
        st["k_pages"], st["v_pages"] = (normal(*shape) * channel).to(dtype), normal(*shape).to(dtype)
    if kind == "attention":
        st["q"], st["out"] = 1.5 * normal(c["seqs"], c["heads"] * hd), torch.empty(c["seqs"], c["heads"] * hd, device="cuda")
    elif kind == "append":
        st["k"], st["v"] = normal(c["n"], kv * hd), (normal(c["n"], kv, hd) * torch.exp(normal(kv, 1))).flatten(1)
        news = _news(c)
        st["start"] = torch.tensor([n - m for n, m in zip(lens, news)], dtype=torch.int32).cuda()
        st["first"] = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32).cuda()
    else:
        st["pool"] = torch.stack([normal(*shape).to(dtype) for _ in range(c["planes"])])
        S = len(lens)
        st["start"] = torch.empty(S, dtype=torch.int32, device="cuda")
        if kind == "branch":
            parents, counts, cut = [0] * S, [0] + [1] * c["branches"], [c["length"]] + [0] * c["branches"]
            st["cut"] = torch.tensor(cut, dtype=torch.int32).cuda()
        else:
            parents, counts = list(range(1, S)) + [NONE], [0] * (S - 1) + [c["length"]]
        st["parents"], st["counts"] = torch.tensor(parents, dtype=torch.int32).cuda(), torch.tensor(counts, dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    return st


# ---- the operators in their plain form -----------------------------------------------------------

def _attend(st):
    c = st["case"]
    S, kv, hd, R = c["seqs"], c["kv"], c["hd"], c["rows"]
    used = _pages(max(_lengths(c)), c)
    at = st["table"][:, :used].long().clamp(min=0)
    k, v = (st[p][at].float().transpose(1, 2).reshape(S, kv, used * R, hd) for p in ("k_pages", "v_pages"))
    seen = torch.arange(used * R, device="cuda") < st["lens"].view(S, 1, 1, 1)
    q = st["q"].view(S, kv, c["heads"] // kv, hd)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = v.masked_fill(~seen.view(S, 1, -1, 1), 0.0)
    st["out"].copy_(torch.matmul(p, v).reshape(S, c["heads"] * hd))


def _append(st):
    c = st["case"]
    token = torch.arange(c["n"], device="cuda")
    seq = (token.unsqueeze(1) >= st["first"][1:]).sum(1)
    row = st["start"][seq] + token - st["first"][seq]
    page = st["table"][seq, row // c["rows"]].long()
    for name, pages in (("k", "k_pages"), ("v", "v_pages")):
        st[pages][page, :, row % c["rows"]] = st[name].view(c["n"], c["kv"], c["hd"]).to(st[pages].dtype)


def _count(refs, entries, by):
    """refs with `by` for each of the entries that name a page."""
    held = entries[entries != NONE].long()
    return refs + by * torch.bincount(held, minlength=refs.numel()).int()


def _fork(st, parents):
    S = st["lens"].numel()
    stays = parents == torch.arange(S, device="cuda")
    held = ((parents >= 0) & (parents < S)).unsqueeze(1)
    from_ = parents.long().clamp(0, S - 1)
    table = torch.where(held, st["table"][from_], NONE)
    refs = _count(_count(st["refs"], st["table"][~stays], -1), table[~stays], 1)
    lens = torch.where(held.squeeze(1), st["lens"][from_], 0)
    st["table"].copy_(table), st["refs"].copy_(refs), st["lens"].copy_(lens)


def _free(st, rows):
    R = st["case"]["rows"]
    goes = torch.arange(st["max_pages"], device="cuda") >= ((rows + R - 1) // R).unsqueeze(1)
    st["refs"].copy_(_count(st["refs"], st["table"][goes], -1))
    st["table"].masked_fill_(goes, NONE)
    st["lens"].copy_(torch.minimum(st["lens"], rows))


def _reserve(st, counts):
    """(what is asked for is there: the cases have pages enough)"""
    R, S, table, lens = st["case"]["rows"], st["lens"].numel(), st["table"], st["lens"]
    one = torch.arange(S, device="cuda")
    last, have, will = (lens // R).long().clamp(max=st["max_pages"] - 1), (lens + R - 1) // R, (lens + counts + R - 1) // R
    page = table[one, last].long()
    writes = (lens % R != 0) & (counts > 0)
    # a page that the writers alone hold stays with the first of them, the others get a copy; one that somebody else holds too is copied for all
    writers = torch.bincount(page[writes], minlength=st["n_pages"])
    first = torch.full((st["n_pages"],), S, device="cuda").scatter_reduce(0, page[writes], one[writes], "amin")
    at = page.clamp(min=0)
    keeps = (writers[at] == st["refs"][at]) & (first[at] == one)
    copies = writes & ~keeps
    need = torch.where(counts > 0, will - have, 0) + copies.int()
    before = torch.cumsum(need, 0) - need
    free = torch.cat([(st["refs"] == 0).nonzero()[:, 0], torch.zeros(1, dtype=torch.int64, device="cuda")])
    j = torch.arange(st["max_pages"], device="cuda")
    new = (j >= have.unsqueeze(1)) & (j < will.unsqueeze(1)) & (counts > 0).unsqueeze(1)
    rank = (before + copies.int() - have).unsqueeze(1) + j
    now = torch.where(new, free[rank.clamp(0, free.numel() - 1)].int(), table)
    own_page = free[before.clamp(max=free.numel() - 1)]
    now[one[copies], last[copies]] = own_page[copies].int()
    st["refs"].copy_(_count(_count(st["refs"], table, -1), now, 1))
    table.copy_(now)
    # the rows in use of every copied page, all planes
    rows_in_use = (torch.arange(R, device="cuda") < (lens % R)[copies].unsqueeze(1)).view(1, -1, 1, R, 1)
    to, from_ = own_page[copies], page[copies]
    st["pool"][:, to] = torch.where(rows_in_use, st["pool"][:, from_], st["pool"][:, to])
    st["start"].copy_(torch.where(counts > 0, lens, NONE))
    lens += counts


def _compact(st):
    used = st["refs"] > 0
    page = torch.arange(st["n_pages"], device="cuda")
    below = page < used.sum()
    to, from_ = (~used & below).nonzero()[:, 0], (used & ~below).nonzero()[:, 0]
    st["pool"][:, to] = st["pool"][:, from_]
    st["refs"][to] = st["refs"][from_]
    st["refs"][from_] = 0
    place = page.int().scatter(0, from_, to.int())
    st["table"].copy_(torch.where(st["table"] != NONE, place[st["table"].long().clamp(min=0)], NONE))


def _sample(st):
    l = st["logits"].double()
    params = st["params"]
    p = params.view(torch.float32)
    t, k, top_p, min_p = p[:, :1].double(), params[:, 1:2], p[:, 2:3].double(), p[:, 3:].double()
    greedy = t <= 0
    t, k = torch.where(greedy, 1.0, t), torch.where(greedy, 1, torch.where(k == 0, l.shape[1], k))
    w = torch.exp((l - l.amax(1, keepdim=True)) / t)
    order = torch.sort(l, dim=1, descending=True, stable=True).indices  # (of equal ones the lower index first)
    rank = torch.arange(l.shape[1], device="cuda")
    falling = w.gather(1, order) * (rank < k)
    before = torch.cumsum(falling, 1) - falling
    kept = ((before < top_p * falling.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0)) & (falling >= min_p) & (rank < k)
    w = w * torch.zeros_like(kept).scatter(1, order, kept)
    upto = torch.cumsum(w, 1)
    mass = upto[:, -1:]
    pick = (upto <= st["u"].double().unsqueeze(1) * mass).sum(1, keepdim=True)
    st["token"].copy_(pick.squeeze(1))
    st["prob"].copy_((w.gather(1, pick) / mass).squeeze(1))


def _run_plain(st):
    kind = st["case"]["kind"]
    if kind == "attention":
        _attend(st)
    elif kind == "append":
        _append(st)
    elif kind == "branch":
        _fork(st, st["parents"])
        _reserve(st, st["counts"])
        _free(st, st["cut"])
    elif kind == "turnover":
        _fork(st, st["parents"])
        _compact(st)
        _reserve(st, st["counts"])
    else:
        _sample(st)


# ---- the framework's ---------------------------------------------------------------------------

_KEPT = {}  # what a program makes once: its context, and one workspace that all its calls share


def _ops():
    if not _KEPT:
        import wick_amd
        from wick_amd import lfm2

        _KEPT.update(lfm2=lfm2, ops=lfm2.Lfm2Ops(wick_amd.RocmContext(0)), scratch=torch.empty(0, dtype=torch.uint8, device="cuda"))
    return _KEPT["ops"], _KEPT["lfm2"]


def _workspace(nbytes):
    if _KEPT["scratch"].numel() < nbytes:
        torch.cuda.synchronize()
        _KEPT["scratch"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return _KEPT["scratch"].data_ptr()


def _handles(st, lfm2):
    """The pool and its table as the calls take them: a program makes them once."""
    if "pages" not in st:
        c = st["case"]
        dtype = {"f32": lfm2.KV_F32, "f16": lfm2.KV_F16}[c["type"]]
        st["dtype"] = dtype
        st["pages"] = lfm2.KvPages(st["table"].data_ptr(), st["lens"].data_ptr(), st["refs"].data_ptr(), n_seqs=st["lens"].numel(), max_pages=st["max_pages"],
                                   n_pages=st["n_pages"], page_rows=c["rows"])
        if "pool" in st:
            plane = st["pool"][0].numel() * st["pool"].element_size()
            st["planes"] = lfm2.KvPlanes(st["pool"].data_ptr(), n_planes=c["planes"], plane_bytes=plane, n_kv_heads=c["kv"], head_dim=c["hd"], kv_dtype=dtype)
    return st["pages"], st.get("planes")


def _run_own(st):
    ops, lfm2 = _ops()
    c, kind = st["case"], st["case"]["kind"]
    if kind == "sample":
        rows, n = c["seqs"], c["n"]
        ops.sample(st["logits"].data_ptr(), n, rows, n, st["params"].data_ptr(), st["u"].data_ptr(), st["token"].data_ptr(), st["prob"].data_ptr(),
                   _workspace(lfm2.sample_scratch_bytes(rows, n)))
        return
    pages, planes = _handles(st, lfm2)
    if kind == "attention":
        width = c["heads"] * c["hd"]
        scratch = _workspace(4 * lfm2.attention_paged_scratch_floats(c["seqs"], c["heads"], c["kv"], c["hd"]))
        ops.encode_attention_paged(pages, st["q"].data_ptr(), width, st["k_pages"].data_ptr(), st["v_pages"].data_ptr(), st["dtype"], st["out"].data_ptr(), width,
                                   scratch, c["heads"], c["kv"], c["hd"])
    elif kind == "append":
        ops.encode_kv_paged_append(pages, st["k"].data_ptr(), st["v"].data_ptr(), c["kv"] * c["hd"], st["k_pages"].data_ptr(), st["v_pages"].data_ptr(), st["dtype"],
                                   st["start"].data_ptr(), c["n"], c["kv"], c["hd"], first=st["first"].data_ptr())
    else:
        moves = _workspace(4 * lfm2.kv_pages_moves_words(pages))
        ops.kv_pages_fork(pages, st["parents"].data_ptr())
        if kind == "turnover":
            ops.kv_pages_compact(pages, moves, planes)
        ops.kv_pages_reserve(pages, st["counts"].data_ptr(), st["start"].data_ptr(), moves, planes)
        if kind == "branch":
            ops.kv_pages_free(pages, st["cut"].data_ptr())


def run(st):
    if own:
        _run_own(st)
    else:
        _run_plain(st)
    kind = st["case"]["kind"]
    names = {"attention": ("out",), "append": ("k_pages", "v_pages"), "sample": ("token", "prob")}.get(kind, ("table", "lens", "refs", "start", "pool"))
    return {name: st[name] for name in names}


# ---- what the outputs should be ----------------------------------------------------------------------

def _exact_pages(st):
    """The pass on lists, page by page."""
    c = st["case"]
    R, S, branch = c["rows"], st["lens"].numel(), c["kind"] == "branch"
    lens = st["lens"].tolist()
    held = [[p for p in row if p != NONE] for row in st["table"].tolist()]
    pool = st["pool"].clone()
    parents, counts = st["parents"].tolist(), st["counts"].tolist()
    held, lens = [list(held[p]) if p >= 0 else [] for p in parents], [lens[p] if p >= 0 else 0 for p in parents]
    if not branch:
        in_use = sorted({p for h in held for p in h})
        holes = [p for p in range(len(in_use)) if p not in set(in_use)]
        new = dict(zip([p for p in in_use if p >= len(in_use)], holes))
        for a, b in new.items():
            pool[:, b] = pool[:, a]
        held = [[new.get(p, p) for p in h] for h in held]
    in_use = {p for h in held for p in h}
    free = (p for p in range(st["n_pages"]) if p not in in_use)
    start, holders = [NONE] * S, {}
    for s in range(S):
        for p in held[s]:
            holders.setdefault(p, []).append(s)
    for s in range(S):
        if not counts[s]:
            continue
        start[s] = lens[s]
        if lens[s] % R:
            p = held[s][lens[s] // R]
            if holders[p][0] != s or not all(counts[h] for h in holders[p]):
                q = next(free)
                pool[:, q, :, :lens[s] % R] = pool[:, p, :, :lens[s] % R]
                held[s][lens[s] // R] = q
        lens[s] += counts[s]
        while len(held[s]) * R < lens[s]:
            held[s].append(next(free))
    return {"table": None, "lens": None, "refs": None, "start": None, "pool": pool}


def exact(case, seed):
    st, c = prepare(case, seed), dict(case)
    kind = c["kind"]
    if kind in ("branch", "turnover"):
        return _exact_pages(st)
    if kind == "append":
        lens, news, token = _lengths(c), _news(c), 0
        table, out = st["table"].cpu().numpy(), {"k_pages": st["k_pages"].double(), "v_pages": st["v_pages"].double()}
        for s, m in enumerate(news):
            for r in range(max(0, lens[s] - m), max(0, lens[s] - m) + m):
                page = int(table[s, r // c["rows"]])
                for name in ("k", "v"):
                    out[name + "_pages"][page, :, r % c["rows"]] = st[name][token].view(c["kv"], c["hd"]).double()
                token += 1
        return out
    if kind == "attention":
        out = torch.empty(c["seqs"], c["heads"], c["hd"], dtype=torch.float64, device="cuda")
        group, table = c["heads"] // c["kv"], st["table"].cpu()
        for s, n in enumerate(_lengths(c)):
            at = table[s, :_pages(n, c)].long().cuda()
            for h in range(c["kv"]):
                k, v = (st[p][at, h].flatten(0, 1)[:n].double() for p in ("k_pages", "v_pages"))
                q = st["q"][s].view(-1, c["hd"])[h * group:(h + 1) * group].double()
                out[s, h * group:(h + 1) * group] = torch.softmax(q @ k.T * c["hd"] ** -0.5, -1) @ v
        return {"out": out.flatten(1)}
    prob = np.empty(c["seqs"])
    logits, u, params = st["logits"].cpu().numpy().astype(np.float64), st["u"].cpu().numpy(), st["params"].cpu().numpy()
    for r in range(c["seqs"]):
        t, top_p, min_p = (float(params[r, i:i + 1].view(np.float32)[0]) for i in (0, 2, 3))
        k = 1 if t <= 0 else int(params[r, 1]) or c["n"]
        x = logits[r]
        order = np.argsort(-x, kind="stable")[:k]
        w = np.exp((x[order] - x[order[0]]) / (t if t > 0 else 1.0))
        if top_p < 1:
            w = w[:1 + int(np.searchsorted(np.cumsum(w), top_p * w.sum()))]
        w = w[w >= min_p]
        index = np.sort(order[:w.size])
        by_index = w[np.argsort(order[:w.size])]
        upto = np.cumsum(by_index)
        at = int(np.searchsorted(upto, float(u[r]) * upto[-1], side="right"))
        assert index.size > at
        prob[r] = by_index[at] / upto[-1]
    return {"token": None, "prob": torch.from_numpy(prob)}


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "sample":
        return {"bytes": 4 * c["seqs"] * c["n"] + 28 * c["seqs"], "flops": 0}
    row = c["kv"] * c["hd"] * TYPES[c["type"]].itemsize  # bytes of a row in one plane
    if c["kind"] == "attention":
        rows = sum(_lengths(c))
        return {"bytes": 2 * rows * row + 8 * c["seqs"] * c["heads"] * c["hd"] + 4 * sum(_pages(n, c) for n in _lengths(c)), "flops": 4 * c["heads"] * c["hd"] * rows}
    if c["kind"] == "append":
        return {"bytes": 2 * c["n"] * (row + 4 * c["kv"] * c["hd"]), "flops": 0}
    pages = _pages(c["length"], c)
    if c["kind"] == "branch":  # the table's rows written, taken back; the last page's rows read once, written for each
        return {"bytes": 8 * c["branches"] * pages + (c["branches"] + 1) * c["planes"] * (c["length"] % c["rows"]) * row, "flops": 0}
    # a session's pages move into the place of the one that left
    return {"bytes": 8 * c["seqs"] * pages + 2 * pages * c["planes"] * c["rows"] * row, "flops": 0}
