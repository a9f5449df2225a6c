"""The operators of paged serving, as cases to be timed and compared.

A serving loop over a paged key/value cache calls five operators besides the packed linears:

  append     RoPE of the new rows' q and k, and k and v into their pages
  attention  each row's query heads over positions 0 .. pos of its sequence's pages
  fork       sequences take over other sequences' pages (beam search, n-best sampling), and each gets a page of
             its own to write its next token to (the page is copied where it is shared)
  compact    the pages in use move to the front of the pool
  logprobs   log probabilities of given tokens, the entropy, and the top alternatives of rows of logits

``run`` computes them with elementary torch operations where ``own`` is false, and with the package's own calls
where it is true.  A cache holds [layers][pages][page][kv heads][head dim] 16-bit values; ``table[s][j]`` is the
page of positions j * page .. of sequence s, -1 for none, and ``refs[p]`` says how many table entries name page p.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MIN_TEMPERATURE = 1e-4  # the sampler's floor


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user, one token: the paged form of the batch-1 decode step (32 query / 8 kv heads), where latency counts
        dict(name="attn_one_row", op="attention", rows=1, per_seq=1, idle=0, heads=32, kv_heads=8, head_dim=128,
             shortest=1537, longest=1537, page=16, type="f16"),
        # a lockstep batch of 16 with one kv head per query head, caches near 2048 entries, stacked q/k/v rows
        dict(name="attn_batch_mha", op="attention", rows=16, per_seq=1, idle=0, heads=32, kv_heads=32, head_dim=64,
             shortest=1025, longest=2047, page=64, type="f16"),
        # continuous batching: 64 slots, lengths from 1 to 8191, some slots empty
        dict(name="attn_ragged_long", op="attention", rows=64, per_seq=1, idle=3, heads=32, kv_heads=8, head_dim=128,
             shortest=1, longest=8191, page=16, type="bf16"),
        # a chunk of a prompt: 128 consecutive tokens of one sequence, each over what came before it (12 / 2 heads)
        dict(name="attn_chunk", op="attention", rows=128, per_seq=128, idle=0, heads=12, kv_heads=2, head_dim=128,
             shortest=1152, longest=1152, page=16, type="f16"),
        # the append of a batch-1 step
        dict(name="append_one_row", op="append", rows=1, per_seq=1, idle=0, heads=32, kv_heads=8, head_dim=128,
             shortest=100, longest=100, page=16, type="f16"),
        # the append of a full batch, q, k and v read from one linear's stacked rows, some slots empty
        dict(name="append_batch", op="append", rows=128, per_seq=1, idle=5, heads=32, kv_heads=32, head_dim=64,
             shortest=1, longest=255, page=32, type="bf16"),
        # one beam search step of 4 beams on a 28-layer cache
        dict(name="fork_beams", op="fork", groups=1, beams=4, layers=28, kv_heads=2, head_dim=128, length=701,
             page=16, type="f16"),
        # 16 beam searches at once on a 32-layer cache
        dict(name="fork_batch", op="fork", groups=16, beams=4, layers=32, kv_heads=8, head_dim=128, length=505,
             page=16, type="f16"),
        # a small pool tidied up after some sequences have left
        dict(name="compact_small", op="compact", seqs=7, blocks=9, pages=150, layers=24, kv_heads=4, head_dim=64,
             page=16, type="bf16"),
        # a large pool, a bit more than half in use, before it is made smaller
        dict(name="compact_large", op="compact", seqs=32, blocks=40, pages=2311, layers=28, kv_heads=2, head_dim=128,
             page=16, type="f16"),
        # the token that was just picked, with its five best alternatives
        dict(name="logprobs_one_row", op="logprobs", rows=1, n=32768, top=5, temperature=1.0, pad=0),
        # a prompt's chunk scored token by token over a large vocabulary
        dict(name="logprobs_chunk", op="logprobs", rows=128, n=151936, top=20, temperature=0.7, pad=0),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(32, 8, 128), (32, 32, 64), (12, 2, 128), (15, 5, 64), (16, 2, 64), (8, 1, 128), (6, 6, 128), (7, 7, 32)]


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "fork", "compact", "logprobs"])
    kind = rng.choice(["f16", "bf16"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    page = rng.choice([8, 16, 24, 32, 64, 100])
    if op in ("attention", "append"):
        chunk = op == "attention" and rng.random() < 0.4
        seqs = _log_int(rng, 1, 6 if chunk else 48)
        per = _log_int(rng, 2, 33) if chunk else 1
        most = 4000 if op == "attention" else 300
        longest = _log_int(rng, per, most)
        shortest = _log_int(rng, per, longest)
        idle = 0 if chunk else rng.randint(0, seqs // 4)
        return dict(op=op, rows=seqs * per, per_seq=per, idle=idle, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    shortest=shortest, longest=longest, page=page, type=kind)
    if op == "fork":
        return dict(op=op, groups=_log_int(rng, 1, 12), beams=rng.randint(2, 6), layers=_log_int(rng, 1, 28),
                    kv_heads=min(kv_heads, 8), head_dim=head_dim, length=_log_int(rng, 1, 700), page=min(page, 32),
                    type=kind)
    if op == "compact":
        seqs, blocks = _log_int(rng, 1, 40), _log_int(rng, 1, 24)
        return dict(op=op, seqs=seqs, blocks=blocks, pages=seqs * blocks + _log_int(rng, 1, 600),
                    layers=_log_int(rng, 1, 20), kv_heads=min(kv_heads, 8), head_dim=head_dim, page=min(page, 32),
                    type=kind)
    n = _log_int(rng, 50, 151936)
    return dict(op=op, rows=_log_int(rng, 1, 127), n=n, top=rng.randint(0, 20), temperature=rng.choice([1.0, 0.6, 1.3]),
                pad=rng.choice([0, 3, 64]))


# ------------------------------------------------------------------------------------------------ sizes of a case
def _lengths(c):
    """Positions that each sequence holds, the new ones among them: spread over [shortest, longest] by the golden
    ratio, the first one the longest; 0 for an idle slot (every fifth, from the third on)."""
    seqs = c["rows"] // c["per_seq"]
    lo, hi = c["shortest"], c["longest"]
    out = [hi if i == 0 else round(lo * (hi / lo) ** ((i * 0.6180339887) % 1.0)) for i in range(seqs)]
    for i in range(c["idle"]):
        out[(3 + 5 * i) % seqs] = 0
    return out


def _parents(c):
    """Each group's beams continue its better half: beam i takes over beam i // 2."""
    return [g * c["beams"] + i // 2 for g in range(c["groups"]) for i in range(c["beams"])]


def _in_use(c):
    """Blocks that each sequence of a compaction still holds: every third one has left, others are partly filled."""
    return [0 if s % 3 == 1 else max(1, c["blocks"] - (s * 5) % c["blocks"]) for s in range(c["seqs"])]


def _page_bytes(c):
    return 2 * c["layers"] * c["page"] * c["kv_heads"] * c["head_dim"] * 2  # K and V of all layers


def work(case):
    c = case
    if c["op"] == "attention":
        lens = _lengths(c)
        kv = sum(lens) * c["kv_heads"] * c["head_dim"] * 2 * 2
        rows_len = sum(n - i for n in lens if n for i in range(c["per_seq"]))
        blocks = sum(-(-n // c["page"]) for n in lens)
        return {"bytes": kv + 2 * c["rows"] * c["heads"] * c["head_dim"] * 4 + 4 * blocks + 8 * c["rows"],
                "flops": 4 * rows_len * c["heads"] * c["head_dim"]}
    if c["op"] == "append":
        rows = sum(1 for n in _lengths(c) if n)
        q, k = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        return {"bytes": rows * (8 * q + 8 * k + 4 * k + 4 * c["head_dim"] + 12), "flops": rows * 3 * (q + k)}
    if c["op"] == "fork":
        seqs, blocks = c["groups"] * c["beams"], -(-c["length"] // c["page"])
        copies = seqs - len(set(_parents(c)))
        return {"bytes": 2 * copies * _page_bytes(c) + 8 * seqs * blocks + 8 * _fork_pages(c), "flops": 0}
    if c["op"] == "compact":
        live, moves = _compact_plan(c)[1:]
        return {"bytes": 2 * moves * _page_bytes(c) + 8 * c["seqs"] * c["blocks"] + 8 * c["pages"], "flops": 0}
    return {"bytes": c["rows"] * (4 * c["n"] + 12 + 8 * c["top"]), "flops": 5 * c["rows"] * c["n"]}


def _fork_pages(c):
    """Pages of a fork's pool: the shared blocks of each group, the beams' own last pages, and as many spare ones."""
    full = (c["length"] - 1) // c["page"]
    return c["groups"] * full + 3 * c["groups"] * c["beams"]


def _compact_plan(c):
    """Pages of the table's entries (sequence by sequence), pages in use, and pages that have to move: the same
    for every seed, since how much moves is part of what the case stands for."""
    order = list(range(c["pages"]))
    random.Random(7 * c["pages"] + c["seqs"]).shuffle(order)
    live = sum(_in_use(c))
    return order[:live], live, sum(1 for p in order[:live] if p >= live)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def ints(v, shape=None):
        t = torch.tensor(v, dtype=torch.int32, device="cuda")
        return t if shape is None else t.reshape(shape)

    if c["op"] == "logprobs":
        rows, n = c["rows"], c["n"]
        # a model's logits: wide, a few tokens far ahead, some ruled out
        x = randn(rows, n + c["pad"]) * 2.5
        x[:, :n] += 9.0 * (torch.rand(rows, n, generator=g, device="cuda") < 4.0 / n)
        x[:, :n].masked_fill_(torch.rand(rows, n, generator=g, device="cuda") < 0.001, -math.inf)
        s["logits"] = x[:, :n]
        s["ids"] = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
        k = min(c["top"], n)
        s["logprob"], s["entropy"] = (torch.empty(rows, device="cuda") for _ in range(2))
        s["top_ids"] = torch.empty(rows, k, device="cuda", dtype=torch.int32)
        s["top_logprobs"] = torch.empty(rows, k, device="cuda")
        if own:
            from gsdlq_b200 import ops
            s["job"] = ops.logprobs_job(s["logits"], ids=s["ids"], logprob=s["logprob"], entropy=s["entropy"],
                                        top_ids=s["top_ids"], top_logprobs=s["top_logprobs"],
                                        temperature=c["temperature"])
        return s

    ps, nkv, hd = c["page"], c["kv_heads"], c["head_dim"]
    if c["op"] in ("attention", "append"):
        lens, layers = _lengths(c), 1
        blocks = [-(-n // ps) for n in lens]
        n_pages, max_blocks = sum(blocks) + 5, max(blocks) + 2
        perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
        table, at = [], 0
        for b in blocks:
            table.append(perm[at:at + b] + [-1] * (max_blocks - b))
            at += b
        used = perm[:at]
        refs = [0] * n_pages
        for p in used:
            refs[p] = 1
    elif c["op"] == "fork":
        layers, n_pages = c["layers"], _fork_pages(c)
        full, seqs = (c["length"] - 1) // ps, c["groups"] * c["beams"]
        perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
        table, refs, max_blocks = [], [0] * n_pages, full + 2
        for i in range(seqs):
            shared = perm[(i // c["beams"]) * full:(i // c["beams"] + 1) * full]
            last = perm[c["groups"] * full + i]
            table.append(shared + [last, -1])
            for p in shared + [last]:
                refs[p] += 1
    else:
        layers, n_pages, max_blocks = c["layers"], c["pages"], c["blocks"]
        used = _compact_plan(c)[0]
        table, refs, at = [], [0] * n_pages, 0
        for b in _in_use(c):
            table.append(used[at:at + b] + [-1] * (max_blocks - b))
            at += b
        for p in used:
            refs[p] = 1

    dt = TYPES[c["type"]]
    # keys carry a bias per channel, as rotated keys do; values are centred
    s["k"] = randn(layers, n_pages, ps, nkv, hd, dtype=dt)
    s["k"] += 0.5 * randn(nkv, hd, dtype=dt)
    s["v"] = randn(layers, n_pages, ps, nkv, hd, dtype=dt)
    s["table"], s["refs"] = ints(table, (len(table), max_blocks)), ints(refs)
    kv = None
    if own:
        from gsdlq_b200 import ops, paged
        kv = s["kv"] = paged.PagedKV.wrap(s["k"], s["v"], s["table"], s["refs"])

    if c["op"] in ("attention", "append"):
        rows, heads, per = c["rows"], c["heads"], c["per_seq"]
        pos = [n - per + i if n else -1 for n in lens for i in range(per)]
        s["pos"] = ints(pos)
        s["row_seq"] = ints([r // per for r in range(rows)]) if per > 1 else None
        # q, k and v as column ranges of one linear's output rows
        qkv = randn(rows, (heads + 2 * nkv) * hd)
        s["q"] = qkv[:, :heads * hd].unflatten(1, (heads, hd))
        s["new_k"] = qkv[:, heads * hd:(heads + nkv) * hd].unflatten(1, (nkv, hd))
        s["new_v"] = qkv[:, (heads + nkv) * hd:].unflatten(1, (nkv, hd))
        s["q"] *= 1.5
        s["out"] = torch.empty(rows, heads, hd, device="cuda")
    if c["op"] == "attention" and own:
        s["job"] = ops.paged_attn_job(kv, 0, s["q"], s["out"], s["pos"], sm_scale=1.0 / math.sqrt(hd),
                                      work=ops.attention_paged_work(kv, rows, heads), row_seq=s["row_seq"])
    if c["op"] == "append":
        angle = torch.arange(c["longest"], dtype=torch.float64)[:, None] * 1e6 ** (
            -torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
        s["rope"] = torch.stack((angle.cos(), angle.sin()), -1).float().cuda()
        if own:
            s["job"] = ops.paged_append_job(kv, 0, s["q"], s["new_k"], s["new_v"], s["out"], s["pos"], s["rope"],
                                            row_seq=s["row_seq"])
    if c["op"] == "fork":
        s["parent"] = ints(_parents(c))
        s["pos"] = ints([c["length"] - 1] * seqs)
    if c["op"] == "compact":
        # what the pass starts from: a second pass on the same state has the same pages to move
        s["table0"], s["refs0"] = s["table"].clone(), s["refs"].clone()
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _attention(s):
    c, ps = s["case"], s["case"]["page"]
    rows, nkv, hd = c["rows"], c["kv_heads"], c["head_dim"]
    t = torch.arange(c["longest"], device="cuda")
    table = s["table"] if s["row_seq"] is None else s["table"][s["row_seq"].long()]
    slot = table[:, t // ps].long().clamp_min(0) * ps + t % ps
    k = s["k"][0].reshape(-1, nkv, hd)[slot].float()
    v = s["v"][0].reshape(-1, nkv, hd)[slot].float()
    q = s["q"].reshape(rows, nkv, -1, hd)
    x = torch.einsum("rghd,rtgd->rght", q, k) * (1.0 / math.sqrt(hd))
    x = x.masked_fill(t > s["pos"][:, None, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m.masked_fill(m == -math.inf, 0.0))
    out = torch.einsum("rght,rtgd->rghd", e, v) / e.sum(-1, keepdim=True)
    return out.masked_fill(s["pos"][:, None, None, None] < 0, 0.0).reshape(rows, -1, hd)


def _append(s):
    ps = s["case"]["page"]
    row = (s["pos"] >= 0).nonzero()[:, 0]
    pos = s["pos"][row].long()
    slot = s["table"][row, pos // ps].long() * ps + pos % ps
    cos, sin = (s["rope"][pos][:, None, :, i] for i in range(2))

    def rotate(x):
        a, b = x[row, :, 0::2], x[row, :, 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    for_k, for_v = s["k"][0].flatten(0, 1), s["v"][0].flatten(0, 1)
    for_k[slot] = rotate(s["new_k"]).to(for_k.dtype)
    for_v[slot] = s["new_v"][row].to(for_v.dtype)
    s["out"].copy_(s["q"])
    s["out"][row] = rotate(s["q"])
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _count(table, n_pages):
    """How many entries of a table name each page."""
    e = table.reshape(-1).long()
    return torch.zeros(n_pages + 1, dtype=torch.int32, device=e.device).index_add_(
        0, torch.where(e >= 0, e, n_pages), torch.ones_like(e, dtype=torch.int32))[:n_pages]


def _fork(s):
    table, refs, ps = s["table"], s["refs"], s["case"]["page"]
    parent = s["parent"].long()
    taken = torch.where(parent[:, None] >= 0, table[parent.clamp_min(0)], -1)
    refs += _count(taken, refs.numel()) - _count(table, refs.numel())
    table.copy_(taken)
    # a page to write to for every sequence: row by row, the one it has unless others hold it too (then a copy,
    # the last holder in the list keeps it), or a new one; new pages are the free ones in their order
    row = torch.arange(table.shape[0], device="cuda")
    block = s["pos"].long() // ps
    page = table[row, block]
    before = ((page[None, :] == page[:, None]) & (row[None, :] < row[:, None])).sum(1)
    shared = (page >= 0) & (refs[page.long().clamp_min(0)] - before > 1)
    need = shared | (page < 0)
    free = torch.sort((refs <= 0).to(torch.int32), descending=True, stable=True).indices
    new = torch.where(need, free[(need.cumsum(0) - 1).clamp_min(0)], page.long())
    src, dst = page[shared].long(), new[shared]
    refs.index_add_(0, src, torch.full_like(src, -1, dtype=torch.int32))
    refs[new[need]] = 1
    table[row, block] = new.int()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"table": table, "refs": refs, "k": s["k"], "v": s["v"]}


def _compact(s):
    table, refs = s["table"], s["refs"]
    live = refs > 0
    n = live.sum()
    page = torch.arange(refs.numel(), device="cuda")
    dst = (~live & (page < n)).nonzero()[:, 0]
    src = (live & (page >= n)).nonzero()[:, 0].flip(0)
    to = page.int()
    to[src] = dst.int()
    table.copy_(torch.where(table >= 0, to[table.long().clamp_min(0)], table))
    refs[dst] = refs[src]
    refs[src] = 0
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"table": table, "refs": refs, "k": s["k"], "v": s["v"]}


def _logprobs(s):
    c = s["case"]
    x = torch.nan_to_num(s["logits"], nan=-1e4, posinf=100.0, neginf=-1e4) / max(c["temperature"], MIN_TEMPERATURE)
    u = x - x.amax(1, keepdim=True)
    e = torch.exp(u)
    total = e.sum(1, keepdim=True)
    lp = u - torch.log(total)
    top = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :min(c["top"], c["n"])]
    return {"logprob": lp.gather(1, s["ids"].long()[:, None])[:, 0],
            "entropy": (torch.log(total) - (e * u).sum(1, keepdim=True) / total)[:, 0],
            "top_ids": top.int(), "top_logprobs": lp.gather(1, top)}


def run(state):
    s, op = state, state["case"]["op"]
    if op == "compact":  # back to the pool as it was before the pass
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
    if not own:
        return {"attention": _attention, "append": _append, "fork": _fork, "compact": _compact,
                "logprobs": _logprobs}[op](s)
    from gsdlq_b200 import ops
    if op == "attention":
        ops.attention_paged(s["job"])
        return s["out"]
    if op == "append":
        ops.rope_kv_paged(s["job"])
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if op == "logprobs":
        ops.logprobs_rows(s["job"])
        return {"logprob": s["logprob"], "entropy": s["entropy"], "top_ids": s["top_ids"],
                "top_logprobs": s["top_logprobs"]}
    if op == "fork":
        s["kv"].fork(s["parent"])
        s["kv"].reserve(s["pos"])
    else:
        s["kv"].compact()
    return {"table": s["table"], "refs": s["refs"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    c = dict(case)
    if c["op"] in ("fork", "compact"):
        return None  # nothing is computed but whole numbers, the rest is copied
    s = prepare(c, seed)
    if c["op"] == "logprobs":
        z = s["logits"].double()
        z = torch.where(z.isnan() | (z == -math.inf), -1e4, torch.where(z == math.inf, 100.0, z))
        z /= max(c["temperature"], MIN_TEMPERATURE)
        norm = torch.logsumexp(z, 1)
        p = torch.exp(z - norm[:, None])
        best = torch.topk(z, min(c["top"], c["n"]), dim=1).values
        return {"logprob": z[torch.arange(c["rows"]), s["ids"].long()] - norm,
                "entropy": -(p * (z - norm[:, None])).sum(1), "top_ids": None, "top_logprobs": best - norm[:, None]}
    pos, table, ps = s["pos"].tolist(), s["table"].tolist(), c["page"]
    seq = range(c["rows"]) if s["row_seq"] is None else s["row_seq"].tolist()
    if c["op"] == "attention":
        out = torch.zeros(c["rows"], c["heads"], c["head_dim"], dtype=torch.float64, device="cuda")
        group = c["heads"] // c["kv_heads"]
        for r, last in enumerate(pos):
            if last < 0:
                continue
            pages = torch.tensor(table[seq[r]][:last // ps + 1], device="cuda")
            k, v = (s[x][0, pages].flatten(0, 1)[:last + 1].double().repeat_interleave(group, 1) for x in "kv")
            w = torch.softmax((k * s["q"][r].double()).sum(-1) / math.sqrt(c["head_dim"]), 0)
            out[r] = (w[..., None] * v).sum(0)
        return out
    k, v, q = s["k"].double(), s["v"].double(), s["q"].double().clone()
    for r, at in enumerate(pos):
        if at < 0:
            continue
        turn = torch.complex(*s["rope"][at].double().unbind(-1))
        p = table[seq[r]][at // ps]
        q[r] = torch.view_as_real(torch.view_as_complex(q[r].unflatten(-1, (-1, 2))) * turn).flatten(-2)
        nk = s["new_k"][r].double().unflatten(-1, (-1, 2)).contiguous()
        k[0, p, at % ps] = torch.view_as_real(torch.view_as_complex(nk) * turn).flatten(-2)
        v[0, p, at % ps] = s["new_v"][r].double()
    return {"q": q, "k": k, "v": v}
