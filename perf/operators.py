"""What is measured of the decoding operators: page moves of the paged key-value cache (fork,
compact, extend), attention of new tokens over that cache (decode: one token a sequence; window:
many, causal, with a sliding window and first tokens that stay visible) and beam search's
selection.  Each has a plain form in elementary torch operations and the framework's call."""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
INF = float("inf")


# ---- cases -----------------------------------------------------------------------------------
def listed():
    return [
        # one prompt's four beams after a step, a small model: launch latency decides
        dict(name="fork_small", op="fork", groups=1, beams=4, survivors=2, layers=2, kv_heads=4, head_dim=64, page=16,
             min_len=20, max_len=200, pages=96, dtype="f16"),
        # a serving batch of beam searches, every group's last pages copied for the repeated parents
        dict(name="fork_serving", op="fork", groups=16, beams=8, survivors=3, layers=8, kv_heads=8, head_dim=128, page=64,
             min_len=500, max_len=1000, pages=800, dtype="bf16"),
        # half of a pool's pages in use, scattered: moved together before the pool is shrunk or saved
        dict(name="compact", op="compact", groups=36, beams=1, survivors=1, layers=8, kv_heads=8, head_dim=128, page=64,
             min_len=700, max_len=1100, pages=1200, dtype="bf16"),
        # chunks of ragged prompts enter the cache: pages taken, keys and values of one layer written
        dict(name="extend", op="extend", seqs=16, min_len=0, max_len=700, min_new=1, max_new=512, kv_heads=8, head_dim=128,
             page=16, pages=1400, dtype="bf16"),
        # one user's next token after a short prompt
        dict(name="decode_one", op="decode", seqs=1, min_len=203, max_len=203, q_heads=32, kv_heads=8, head_dim=128, page=16,
             window=0, sinks=0, dtype="f16"),
        # a stream of chats under a sliding window whose first tokens stay visible
        dict(name="decode_window", op="decode", seqs=48, min_len=1, max_len=5000, q_heads=28, kv_heads=4, head_dim=64, page=32,
             window=1000, sinks=4, dtype="f16"),
        # a serving batch with long and short contexts, the 64 / 8 heads of the benchmark's decoder layer
        dict(name="decode_serving", op="decode", seqs=64, min_len=100, max_len=16000, q_heads=64, kv_heads=8, head_dim=128,
             page=64, window=0, sinks=0, dtype="bf16"),
        # a few drafted tokens are checked at once
        dict(name="window_draft", op="window", seqs=3, min_new=1, max_new=9, min_past=30, max_past=700, q_heads=16, kv_heads=4,
             head_dim=64, page=16, window=256, sinks=4, dtype="f16"),
        # ragged prompts' chunks over what is cached, sliding window and sinks
        dict(name="window_chunks", op="window", seqs=4, min_new=300, max_new=2000, min_past=0, max_past=1500, q_heads=32,
             kv_heads=8, head_dim=128, page=32, window=1024, sinks=4, dtype="bf16"),
        # one long prompt, every earlier token visible
        dict(name="window_prompt", op="window", seqs=1, min_new=8192, max_new=8192, min_past=0, max_past=0, q_heads=64,
             kv_heads=8, head_dim=128, page=64, window=0, sinks=0, dtype="bf16"),
        # one search of four beams over a 32000-token vocabulary
        dict(name="beam_one", op="beam", batch=1, beams=4, vocab=32000, n=4, finished=0, dtype="f32"),
        # a batch of searches over a large vocabulary, twice as many candidates as beams, some beams ended
        dict(name="beam_serving", op="beam", batch=32, beams=8, vocab=128000, n=16, finished=1, dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["fork", "compact", "extend", "decode", "decode", "window", "window", "beam", "beam"])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]))
    if op in ("fork", "compact"):
        c["groups"], c["beams"] = log(1, 16), rng.randint(1, 8) if op == "fork" else 1
        if op == "compact":
            c["groups"] = log(1, 36)
        c["survivors"] = rng.randint(1, c["beams"])
        c["layers"], c["kv_heads"], c["head_dim"] = rng.randint(1, 8), rng.randint(1, 8), rng.choice([64, 80, 96, 128])
        c["page"] = rng.choice([16, 32, 64])
        c["max_len"] = log(50, 1000)
        c["min_len"] = rng.randint(1, c["max_len"])
        most = -(-c["max_len"] // c["page"])
        c["pages"] = c["groups"] * c["beams"] * (most + 1) + rng.randint(8, 100)
        if op == "compact":
            c["pages"] = int(c["pages"] * rng.uniform(1.0, 2.0))
    elif op == "extend":
        c["seqs"], c["kv_heads"], c["head_dim"] = log(1, 16), rng.randint(1, 8), rng.choice([64, 80, 96, 128])
        c["page"], c["min_len"], c["max_len"] = rng.choice([16, 32, 64]), 0, log(1, 700)
        c["max_new"] = log(1, 512)
        c["min_new"] = rng.randint(0, c["max_new"])
        c["pages"] = c["seqs"] * (-(-(c["max_len"] + c["max_new"]) // c["page"]) + 1) + rng.randint(0, 50)
    elif op == "decode":
        c["kv_heads"], c["head_dim"] = rng.randint(1, 8), rng.choice([64, 64, 80, 128, 128, 128])
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 7, 8])
        c["seqs"], c["max_len"], c["page"] = log(1, 64), log(16, 16000), rng.choice([16, 32, 64, 128])
        c["min_len"] = rng.randint(0, c["max_len"])
        c["window"] = rng.choice([0, 0, log(1, 4000)])
        c["sinks"] = rng.choice([0, 4, rng.randint(1, 70)]) if c["window"] else 0
    elif op == "window":
        c["kv_heads"], c["head_dim"] = rng.randint(1, 8), rng.choice([64, 64, 80, 128, 128, 128])
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
        c["seqs"], c["page"] = log(1, 6), rng.choice([16, 32, 64, 128])
        c["max_new"], c["max_past"] = log(1, 2500), rng.choice([0, log(10, 1500)])
        c["min_new"], c["min_past"] = rng.randint(0, c["max_new"]), rng.randint(0, c["max_past"])
        c["window"] = rng.choice([0, log(1, 2000)])
        c["sinks"] = rng.choice([0, 4, rng.randint(1, 200)]) if c["window"] else 0
    else:
        c["dtype"] = rng.choice(["f16", "bf16", "f32"])
        c["beams"], c["vocab"] = rng.randint(1, 8), log(5000, 128000)
        c["batch"] = log(1, 32 if c["dtype"] != "f32" else 16)
        c["n"], c["finished"] = rng.randint(1, 16), rng.randint(0, 1)
    return c


# ---- inputs ----------------------------------------------------------------------------------
def _pools(gen, layers, pages, heads, page, dim, dtype):
    shape = (layers, pages, heads, page, dim)
    return [torch.randn(shape, generator=gen, device=DEV, dtype=dtype) for _ in range(2)]


def _lengths(count, lo, hi, salt=0):
    """A case's `count` lengths of lo..hi, the longest among them: a seed only puts them into another order."""
    n = np.random.RandomState(1000003 * salt + 1009 * count + hi).randint(lo, hi + 1, count).astype(np.int32)
    n[-1] = hi
    return n


def _tables(rs, lengths, shared, beams, page, pages, width):
    """Page table, reference counts: `beams` rows a group share the group's first shared[g] pages and own
    the rest; page numbers in no order."""
    table = np.full((len(lengths) * beams, width), -1, np.int32)
    order, at = rs.permutation(pages).astype(np.int32), 0
    for g, n in enumerate(lengths):
        used = -(-int(n) // page)
        own_pages = used - int(shared[g])
        rows = table[g * beams:(g + 1) * beams]
        rows[:, :shared[g]] = order[at:at + shared[g]]
        at += int(shared[g])
        rows[:, shared[g]:used] = order[at:at + beams * own_pages].reshape(beams, own_pages)
        at += beams * own_pages
    count = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    return table, count


def _on(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrays]


def prepare(case, seed):
    c, op, dt = case, case["op"], TYPES[case["dtype"]]
    rs = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if op in ("fork", "compact"):
        page = c["page"]
        lengths = rs.permutation(_lengths(c["groups"], c["min_len"], c["max_len"]))
        shared = (lengths * 3 // 4) // page if c["beams"] > 1 else lengths * 0  # the prompt's whole pages
        width = -(-c["max_len"] // page) + 1
        table, count = _tables(rs, lengths, shared, c["beams"], page, c["pages"], width)
        s["table"], s["lengths"], s["refcount"] = _on(table, np.repeat(lengths, c["beams"]), count)
        s["k"], s["v"] = _pools(gen, c["layers"], c["pages"], c["kv_heads"], page, c["head_dim"], dt)
        if op == "fork":
            parents = []
            for g in range(c["groups"]):  # `survivors` parents, some of them several times, in no order
                alive = rs.permutation(c["beams"])[:c["survivors"]]
                again = alive[rs.randint(0, c["survivors"], c["beams"] - c["survivors"])]
                parents.append(g * c["beams"] + rs.permutation(np.concatenate([alive, again])))
            s["parents"] = _on(np.concatenate(parents).astype(np.int32))[0]
    elif op == "extend":
        page = c["page"]
        lengths = rs.permutation(_lengths(c["seqs"], c["min_len"], c["max_len"]))
        new = rs.permutation(_lengths(c["seqs"], c["min_new"], c["max_new"], 1))
        width = -(-(c["max_len"] + c["max_new"]) // page)
        table, count = _tables(rs, lengths, lengths * 0, 1, page, c["pages"], width)
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        s["table"], s["lengths"], s["refcount"], s["new"], s["cu"] = _on(table, lengths, count, new, cu)
        s["k"], s["v"] = _pools(gen, 1, c["pages"], c["kv_heads"], page, c["head_dim"], dt)
        for name in ("k_new", "v_new"):
            s[name] = torch.randn(int(cu[-1]), c["kv_heads"], c["head_dim"], generator=gen, device=DEV, dtype=dt)
    elif op in ("decode", "window"):
        page = c["page"]
        if op == "decode":
            lengths = rs.permutation(_lengths(c["seqs"], c["min_len"], c["max_len"]))
            width, rows = max(1, -(-c["max_len"] // page)), c["seqs"]
        else:
            at = rs.permutation(c["seqs"])
            new = _lengths(c["seqs"], c["min_new"], c["max_new"], 1)[at]
            lengths = new + _lengths(c["seqs"], c["min_past"], c["max_past"], 2)[at]
            cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
            width, rows = max(1, -(-(c["max_new"] + c["max_past"]) // page)), int(cu[-1])
            s["cu"] = _on(cu)[0]
        pages = int((-(-lengths // page)).sum()) + 8
        table, _ = _tables(rs, lengths, lengths * 0, 1, page, pages, width)
        s["table"], s["lengths"] = _on(table, lengths)
        k, v = _pools(gen, 1, pages, c["kv_heads"], page, c["head_dim"], dt)
        s["k"], s["v"] = k[0], v[0]
        s["q"] = torch.randn(rows, c["q_heads"], c["head_dim"], generator=gen, device=DEV, dtype=dt)
    else:
        shape = (c["batch"], c["beams"])
        # logits of a language model: a broad body and a few likely tokens
        x = torch.randn(*shape, c["vocab"], generator=gen, device=DEV).mul_(2.0)
        hot = torch.randint(0, c["vocab"], (*shape, 24), generator=gen, device=DEV)
        x.scatter_add_(2, hot, torch.rand(*shape, 24, generator=gen, device=DEV) * 9 + 3)
        s["logits"] = x.to(dt)
        s["scores"] = torch.rand(shape, generator=gen, device=DEV).mul_(-8.0).cumsum(-1)
        s["finished"] = torch.from_numpy(rs.rand(*shape) < 0.25).to(DEV) if c["finished"] else None
    return s


# ---- plain forms -----------------------------------------------------------------------------
def _plain_fork(s):
    k, v, table, lengths, count, parents = (s[n] for n in ("k", "v", "table", "lengths", "refcount", "parents"))
    rows, width = table.shape
    pages, page = k.shape[1], k.shape[3]
    col, row = torch.arange(width, device=DEV), torch.arange(rows, device=DEV)
    live, par = parents >= 0, parents.clamp(min=0).long()
    n = torch.where(live, lengths[par], 0)
    used, fill = (n + page - 1) // page, n % page
    new = torch.where(col < used[:, None], table[par], -1)
    first = torch.full((rows,), rows, device=DEV).scatter_reduce(0, par, torch.where(live, row, rows), "amin")
    dup = live & (fill > 0) & (row != first[par])  # the first child keeps the part-filled page, the others copy it
    last = (used - 1).clamp(min=0).long()
    src = new[row, last].long()
    old = torch.where(col < ((lengths + page - 1) // page)[:, None], table, -1)
    kept = new.clone()
    kept[dup, last[dup]] = -1
    one = torch.ones(rows * width, device=DEV, dtype=torch.int32)
    count = torch.cat([count, count.new_zeros(1)])  # the extra place takes the absent entries
    count.scatter_add_(0, torch.where(old < 0, pages, old).long().reshape(-1), -one)
    count.scatter_add_(0, torch.where(kept < 0, pages, kept).long().reshape(-1), one)
    count = count[:pages]
    fresh = (count == 0).nonzero().reshape(-1)[:int(dup.sum())]  # lowest free pages, in row order
    new[dup, last[dup]] = fresh.int()
    count[fresh] = 1
    rowmask = (torch.arange(page, device=DEV) < fill[dup][:, None])[None, :, None, :, None]
    k[:, fresh] = torch.where(rowmask, k[:, src[dup]], k[:, fresh])
    v[:, fresh] = torch.where(rowmask, v[:, src[dup]], v[:, fresh])
    return new, n.int(), count, k, v


def _plain_compact(s):
    k, v, table, lengths, count = (s[n] for n in ("k", "v", "table", "lengths", "refcount"))
    pages, page = k.shape[1], k.shape[3]
    total = (count > 0).sum()
    at = torch.arange(pages, device=DEV)
    src = ((count > 0) & (at >= total)).nonzero().reshape(-1)
    dst = ((count == 0) & (at < total)).nonzero().reshape(-1)
    to = at.clone()
    to[src] = dst
    valid = torch.arange(table.shape[1], device=DEV) < ((lengths + page - 1) // page)[:, None]
    new = torch.where(valid & (table >= 0), to[table.clamp(min=0).long()], -1).int()
    after = count.clone()
    after[dst], after[src] = count[src], 0
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    return new, after, total.int().reshape(1), k, v


def _positions(cu, total):
    """Sequence of each packed row, and its place in that sequence's new tokens."""
    row = torch.arange(total, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return seq, row - cu[seq]


def _plain_extend(s):
    k, v, table, lengths, count, add = (s[n] for n in ("k", "v", "table", "lengths", "refcount", "new"))
    page = k.shape[3]
    n = lengths + add
    col = torch.arange(table.shape[1], device=DEV)
    had, has = ((lengths + page - 1) // page)[:, None], ((n + page - 1) // page)[:, None]
    want = (col >= had) & (col < has)
    fresh = (count == 0).nonzero().reshape(-1)[:int(want.sum())]  # lowest free pages, in row and then column order
    new = torch.where(col < had, table, -1)
    new[want] = fresh.int()
    after = count.clone()
    after[fresh] = 1
    seq, i = _positions(s["cu"], s["k_new"].shape[0])
    pos = (lengths[seq] + i).long()
    at = new[seq, pos // page].long()
    k[0, at, :, pos % page] = s["k_new"]
    v[0, at, :, pos % page] = s["v_new"]
    return new, n.int(), after, k, v


def _gathered(pool, table):
    """(pages, heads, page, dim) by a table (rows, width): (rows, heads, width * page, dim) in 32 bits."""
    got = pool[table.clamp(min=0).long()]
    return got.permute(0, 2, 1, 3, 4).reshape(table.shape[0], pool.shape[1], -1, pool.shape[3]).float()


def _visible(pos, key, n, window, sinks):
    see = (key <= pos) & (key < n)
    return see & ((key > pos - window) | (key < sinks)) if window else see


def _softmax_product(score, see, v):
    score = score.masked_fill_(~see, -INF)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -INF, 0.0, top)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.matmul(v) / torch.where(total == 0, 1.0, total)
    return out, (total.log() + top).squeeze(-1)


def _plain_decode(s):
    c, q = s["case"], s["q"]
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    rows, heads, dim = q.shape
    qg = q.float().view(rows, k.shape[1], -1, dim)
    n = s["lengths"].view(-1, 1, 1, 1)
    see = _visible(n - 1, torch.arange(k.shape[2], device=DEV), n, c["window"], c["sinks"])
    out, lse = _softmax_product(qg.matmul(k.transpose(2, 3)) / math.sqrt(dim), see, v)
    return out.reshape(rows, heads, dim).to(q.dtype), lse.reshape(rows, heads)


def _plain_window(s):
    c, q, cu = s["case"], s["q"], s["cu"]
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    total, heads, dim = q.shape
    seqs, kv, keys = k.shape[:3]
    seq, i = _positions(cu, total)
    padded = q.new_zeros(seqs, c["max_new"], heads, dim, dtype=torch.float32)
    padded[seq, i] = q.float()
    padded = padded.view(seqs, c["max_new"], kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    n = s["lengths"].view(-1, 1, 1)
    pos = (s["lengths"] - (cu[1:] - cu[:-1])).view(-1, 1, 1) + torch.arange(c["max_new"], device=DEV).view(1, -1, 1)
    see = _visible(pos, torch.arange(keys, device=DEV), n, c["window"], c["sinks"])  # (seqs, new, keys)
    score = padded.reshape(seqs, kv, -1, dim).matmul(k.transpose(2, 3)).div_(math.sqrt(dim))
    score = score.view(seqs, kv, heads // kv, c["max_new"], keys)
    out, lse = _softmax_product(score, see[:, None, None], v[:, :, None])
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, c["max_new"], heads, dim)[seq, i]
    return out.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(seqs, c["max_new"], heads)[seq, i]


def _plain_beam(s):
    n = s["case"]["n"]
    x = s["logits"].float()
    x = torch.where(x.isnan(), -INF, x)
    top = x.amax(-1, keepdim=True)
    total = (x - top).exp().sum(-1, keepdim=True)
    best, token = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lower token first
    logp = (best[..., :n] - top) - total.log()
    score, token = s["scores"][..., None] + logp, token[..., :n]
    if s["finished"] is not None:  # an ended beam goes on as it is, with the padding token
        rank = torch.arange(n, device=DEV)
        ended = s["finished"][..., None]
        score = torch.where(ended, torch.where(rank == 0, s["scores"][..., None], -INF), score)
        token = torch.where(ended, 0, token)
    score, at = torch.sort(score.flatten(1), dim=-1, descending=True, stable=True)  # ties: the lower beam first
    score, at = score[:, :n], at[:, :n]
    return score, (at // n).int(), token.flatten(1).gather(1, at).int()


# ---- one pass --------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        return {"fork": _plain_fork, "compact": _plain_compact, "extend": _plain_extend, "decode": _plain_decode,
                "window": _plain_window, "beam": _plain_beam}[op](s)
    if op in ("fork", "compact", "extend"):
        from quipsharp_b200 import kv_cache as kc
        if op == "fork":
            table, lengths, count = kc.fork_pages(s["k"], s["v"], s["table"], s["lengths"], s["refcount"], s["parents"])
            return table, lengths, count, s["k"], s["v"]
        if op == "compact":
            table, count, used = kc.compact_pages(s["k"], s["v"], s["table"], s["lengths"], s["refcount"])
            return table, count, used, s["k"], s["v"]
        table, lengths, count = kc.extend_pages(s["table"], s["lengths"], s["refcount"], s["new"], c["page"])
        kc.write_kv(s["k_new"], s["v_new"], s["k"][0], s["v"][0], table, lengths, s["cu"])
        return table, lengths, count, s["k"], s["v"]
    if op == "beam":
        from quipsharp_b200.beam import beam_select
        return beam_select(s["logits"], s["scores"], c["n"], finished=s["finished"], pad=0)
    from quipsharp_b200 import attention
    if op == "decode":
        return attention.decode_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=c["window"] or None,
                                          sinks=c["sinks"], return_lse=True)
    return attention.window_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["cu"], window=c["window"] or None,
                                      sinks=c["sinks"], return_lse=True)


# ---- what a pass cannot do without -------------------------------------------------------------
def work(case):
    c, op = case, case["op"]
    size = 4 if c["dtype"] == "f32" else 2
    if op == "beam":
        rows = c["batch"] * c["beams"]
        return {"bytes": rows * c["vocab"] * size + rows * 5 + c["batch"] * c["n"] * 12, "flops": 4 * rows * c["vocab"]}
    kv_row = 2 * c["kv_heads"] * c["head_dim"] * size  # one token's keys and values in one layer
    page = c["page"]
    if op in ("fork", "compact"):
        n = _lengths(c["groups"], c["min_len"], c["max_len"]).astype(np.int64)
        used = -(-n // page)
        meta = 8 * c["beams"] * int((used + 1).sum()) + 8 * c["pages"]
        if op == "fork":
            moved = (c["beams"] - c["survivors"]) * int((n % page).sum())
        else:  # a used page lies behind the first `taken` ones with this chance
            taken = int(used.sum())
            moved = taken * (1 - taken / c["pages"]) * page
        return {"bytes": meta + 2 * c["layers"] * moved * kv_row, "flops": 0}
    if op == "extend":
        n, new = _lengths(c["seqs"], c["min_len"], c["max_len"]), _lengths(c["seqs"], c["min_new"], c["max_new"], 1)
        return {"bytes": 2 * int(new.sum()) * kv_row + 8 * c["pages"] + 8 * int((n + new).sum()) / page, "flops": 0}

    def seen(n):  # keys that the token in place n - 1 sees
        if not c["window"]:
            return n
        return np.minimum(n, c["window"]) + np.clip(n - c["window"], 0, c["sinks"])

    if op == "decode":
        n = _lengths(c["seqs"], c["min_len"], c["max_len"]).astype(np.int64)
        rows, pairs = c["seqs"], int(seen(n).sum())
        keys = pairs
    else:
        new = _lengths(c["seqs"], c["min_new"], c["max_new"], 1)
        past = _lengths(c["seqs"], c["min_past"], c["max_past"], 2)
        rows, pairs, keys = int(new.sum()), 0, 0
        for t, p in zip(new.tolist(), past.tolist()):
            pairs += int(seen(np.arange(p + 1, p + t + 1)).sum())
            if t:
                keys += p + t if not c["window"] else min(p + t, t + c["window"] - 1 + c["sinks"])
    q_bytes = rows * c["q_heads"] * (2 * c["head_dim"] * size + 4)
    return {"bytes": keys * kv_row + q_bytes, "flops": 4 * pairs * c["q_heads"] * c["head_dim"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _exact_attention(s, new, past):
    """Sequence by sequence and head by head: softmax over the keys that each row sees."""
    c, q = s["case"], s["q"]
    table, page, dim = s["table"].cpu().tolist(), c["page"], c["head_dim"]
    share = c["q_heads"] // c["kv_heads"]
    outs, lses, at = [], [], 0
    for b, (t, p) in enumerate(zip(new, past)):
        n = t + p
        ids = torch.tensor(table[b][:-(-n // page)], device=DEV, dtype=torch.long)
        qs = q[at:at + t].double()
        at += t
        out = torch.zeros(t, c["q_heads"], dim, device=DEV, dtype=torch.float64)
        lse = torch.full((t, c["q_heads"]), -INF, device=DEV, dtype=torch.float64)
        if n and t:
            key = torch.arange(n, device=DEV)[None, :]
            pos = p + torch.arange(t, device=DEV)[:, None]
            hidden = key > pos
            if c["window"]:
                hidden |= (key <= pos - c["window"]) & (key >= c["sinks"])
            for h in range(c["q_heads"]):
                kh = s["k"][ids, h // share].reshape(-1, dim)[:n].double()
                vh = s["v"][ids, h // share].reshape(-1, dim)[:n].double()
                score = torch.where(hidden, -INF, (qs[:, h] @ kh.T) * dim ** -0.5)
                lse[:, h] = torch.logsumexp(score, -1)
                out[:, h] = torch.softmax(score, -1) @ vh
        outs.append(out)
        lses.append(lse)
    return torch.cat(outs), torch.cat(lses)


def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact", "extend"):
        return None  # page numbers and copies: nothing is computed in floating point
    s = prepare(case, seed)
    if op == "beam":
        n = case["n"]
        logp = torch.log_softmax(s["logits"].double(), -1)
        best = []
        for b in range(case["batch"]):
            total = (s["scores"][b].double()[:, None] + logp[b]).sort(dim=-1, descending=True)[0][:, :n]
            if s["finished"] is not None:
                for k in s["finished"][b].nonzero().reshape(-1).tolist():
                    total[k] = -INF
                    total[k, 0] = s["scores"][b, k].double()
            best.append(total.reshape(-1).sort(descending=True)[0][:n])
        return torch.stack(best), None, None
    lengths = s["lengths"].cpu().tolist()
    if op == "decode":
        rows = [_exact_attention({**s, "q": s["q"][b:b + 1], "table": s["table"][b:b + 1]}, [1], [n - 1])
                if n else (torch.zeros(1, case["q_heads"], case["head_dim"], device=DEV, dtype=torch.float64),
                           torch.full((1, case["q_heads"]), -INF, device=DEV, dtype=torch.float64))
                for b, n in enumerate(lengths)]
        return torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows])
    new = (s["cu"][1:] - s["cu"][:-1]).cpu().tolist()
    return _exact_attention(s, new, [n - t for n, t in zip(lengths, new)])
