"""Workloads of the serving operators: attention of new tokens over a paged key-value cache, the write of their keys and values
into its pages, and the keeping of the pages (room for new tokens, forks, freed sequences, compaction).

A case is one of four kinds.  ``decode``: ``sb_attn_decode`` for the newest tokens of a batch.  ``append``: ``kv_append`` of a
step's or a prefill's keys and values.  ``branch``: some sequences are forked, the forks get room for new tokens, some of the
originals are freed (``kv_fork``, ``kv_extend``, ``kv_free``).  ``compact``: live pages move to the front of a pool with holes
(``kv_compact``).

With ``own`` false ``run`` computes the same in elementary torch operations.

The score distribution decides how far back a query looks (``data``): ``spread`` is a head that spreads its stick over the whole
context (scores around -log of the longest length, no key's weight vanishes), ``local`` has scores around 0: about one bit of
stick is broken off per key and what lies some 110 keys back has weight 0 in 32 bits.  ``mixed``: every other key head is local.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
LOCAL_REACH = 110          # keys until a local head's stick is used up: 126 bits at 1.16 per key


def _decode(**kw):
    return {"kind": "decode", "dtype": "bf16", "heads": 16, "kv_heads": 16, "head_dim": 128, "page": 64, "seqs": 1, "low": 1,
            "high": 1, "new": 1, "data": "spread", "attend_current": False, **kw}


def _append(**kw):
    return {"kind": "append", "dtype": "bf16", "kv_heads": 16, "head_dim": 128, "page": 64, "seqs": 1, "low": 1, "high": 1,
            "prompts": False, **kw}


def _pages(kind, **kw):
    return {"kind": kind, "dtype": "bf16", "layers": 4, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 1, "low": 1,
            "high": 1, **kw}


def listed():
    return [
        # the next token of one short prompt: a single small call, where the call itself is most of the time
        _decode(name="decode_one_prompt", dtype="fp16", heads=8, kv_heads=8, head_dim=64, page=16, low=200, high=200, data="local"),
        # the fp32 configuration the operators are validated on: 4 heads, ragged sequences of up to 512 tokens
        _decode(name="decode_fp32", dtype="fp32", heads=4, kv_heads=4, head_dim=64, page=32, seqs=16, low=64, high=512),
        # a serving batch at the headline heads: 64 sequences of 512 to 4096 tokens, every head with its own keys
        _decode(name="decode_batch", seqs=64, low=512, high=4096),
        # shared key heads, small pages, ragged contexts; half of the heads look back a hundred keys only
        _decode(name="decode_shared_heads", heads=32, kv_heads=8, page=16, seqs=48, low=64, high=16384, data="mixed"),
        # one long context alone on the GPU: all of it for one token
        _decode(name="decode_long_context", heads=16, kv_heads=4, low=131072, high=131072),
        # four drafted tokens verified at once, tokens attending to themselves, a page size that is no power of two
        _decode(name="decode_draft", dtype="fp16", heads=32, kv_heads=8, head_dim=64, page=24, seqs=24, low=200, high=3000, new=4,
                attend_current=True),
        # one step's keys and values of a serving batch
        _append(name="append_step", seqs=64, low=512, high=4096),
        # the keys and values of a packed prefill: 64 prompts, some 34000 tokens
        _append(name="append_prompts", kv_heads=8, seqs=64, low=48, high=2000, prompts=True),
        # a few answers sampled from the same prompts
        _pages("branch", name="branch_small", dtype="fp16", layers=2, head_dim=64, page=16, seqs=4, low=100, high=600),
        # every sequence of a batch forked
        _pages("branch", name="branch_batch", seqs=64, low=300, high=1700),
        # a small pool after a few requests have gone
        _pages("compact", name="compact_small", dtype="fp16", layers=2, head_dim=64, page=16, seqs=6, low=100, high=600),
        # a large one after half of its requests have gone
        _pages("compact", name="compact_pool", seqs=64, low=300, high=1700),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["decode", "decode", "decode", "append", "branch", "compact"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        page = rng.choice([16, 16, 32, 64, 64, 128, 24, 48])
        head_dim = rng.choice([64, 64, 128, 128, 128, 96, 72, 80])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12, 16])
        common = dict(dtype=dtype, page=page, head_dim=head_dim, kv_heads=kv_heads)
        if kind == "decode":
            high = _log_uniform(rng, 20, 131072)
            case = _decode(heads=kv_heads * rng.choice([1, 1, 2, 3, 4, 8]), seqs=_log_uniform(rng, 1, 256), high=high,
                           low=max(1, high // rng.choice([1, 2, 8, 64])), new=rng.choice([1, 1, 1, 1, 2, 3, 5]),
                           data=rng.choice(["spread", "spread", "mixed", "local"]), attend_current=rng.random() < 0.3, **common)
            cost = work({**case, "data": "spread"})
            if cost["bytes"] > 9e8 or cost["flops"] > 1.2e9 or (dtype == "fp32" and cost["flops"] > 6e8):
                continue
        elif kind == "append":
            prompts = rng.random() < 0.5
            high = _log_uniform(rng, 1, 8192)
            case = _append(seqs=_log_uniform(rng, 1, 256), high=high, low=max(1, high // rng.choice([1, 4, 32])), prompts=prompts,
                           **common)
            if work(case)["bytes"] > 4e8 or case["seqs"] * high * kv_heads * head_dim * ESIZE[dtype] > 1.2e9:
                continue
        else:
            high = _log_uniform(rng, 16, 4096)
            case = _pages(kind, layers=rng.choice([1, 2, 4, 8]), seqs=_log_uniform(rng, 2, 200), high=high,
                          low=max(1, high // rng.choice([1, 2, 8])), **common)
            if case["seqs"] * (high + 2 * page) * case["layers"] * kv_heads * head_dim * ESIZE[dtype] > 6e8:
                continue
        return case


def lengths(case):
    """The lengths of a case's sequences, the same for every seed: spread evenly over their logarithm, long and short ones mixed."""
    n, lo, hi = case["seqs"], case["low"], case["high"]
    if n == 1:
        return [hi]
    x = np.exp(np.linspace(math.log(lo), math.log(hi), n))
    return [int(v) for v in np.random.default_rng(1).permutation(np.clip(np.round(x), lo, hi))]


def _page_count(lens, page):
    return [-(-n // page) for n in lens]


def _table(counts, width, pages, seed):
    """A page table whose sequences have their pages all over the pool; -1 behind a sequence's last page."""
    order = np.random.default_rng(seed).permutation(pages)
    table = np.full((len(counts), width), -1, dtype=np.int32)
    at = 0
    for row, count in zip(table, counts):
        row[:count] = order[at:at + count]
        at += count
    return table


# ---- what a program has in hand -----------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"decode": _prepare_decode, "append": _prepare_append, "branch": _prepare_pages, "compact": _prepare_pages}
    return {"case": case, **make[case["kind"]](case, gen, seed)}


def _prepare_decode(case, gen, seed):
    dtype, d, heads, kv = DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    lens = lengths(case)
    counts = _page_count(lens, case["page"])
    pages = sum(counts) + 1
    # <q, k> / sqrt(d) ~ N(-shift^2 sqrt(d), 1 + 2 shift^2) for the heads that spread their stick, N(0, 1) for the local ones
    target = math.log(max(max(lens), 4)) + 0.5
    shift = torch.full((kv,), math.sqrt(target / (math.sqrt(d) - 1)), device="cuda", dtype=dtype)
    if case["data"] == "local":
        shift.zero_()
    elif case["data"] == "mixed":
        shift[1::2] = 0

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    q = normal(case["seqs"], heads, case["new"], d)
    q += shift.repeat_interleave(heads // kv)[None, :, None, None]
    k = normal(pages, kv, case["page"], d)
    k -= shift[None, :, None, None]
    table = _table(counts, max(counts), pages, seed)
    return {"q": q, "k_pages": k, "v_pages": normal(pages, kv, case["page"], d), "page_table": torch.from_numpy(table).cuda(),
            "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}


def _prepare_append(case, gen, seed):
    dtype, d, kv = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    lens = lengths(case)
    counts = _page_count(lens, case["page"])
    pages = sum(counts) + 1

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"k_pages": normal(pages, kv, case["page"], d), "v_pages": normal(pages, kv, case["page"], d),
             "page_table": torch.from_numpy(_table(counts, max(counts), pages, seed)).cuda(),
             "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "cu_seqlens": None}
    if case["prompts"]:      # packed, token-major activations handed over as permuted views, as a projection leaves them
        state["k"], state["v"] = (normal(sum(lens), kv, d).transpose(0, 1) for _ in range(2))
        state["cu_seqlens"] = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    else:
        state["k"], state["v"] = (normal(len(lens), kv, 1, d) for _ in range(2))
    return state


def _prepare_pages(case, gen, seed):
    dtype, d, kv, page, n = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"], case["page"], case["seqs"]
    lens = lengths(case)
    counts = _page_count(lens, page)
    width = -(-(case["high"] + page) // page) + 1
    # twice as many slots as sequences; in the pool, room for the forks' own pages
    pages = sum(counts) + 3 * n + 5
    table = np.full((2 * n, width), -1, dtype=np.int32)
    table[:n] = _table(counts, width, pages, seed)
    seq_lens = np.array(lens + [0] * n, dtype=np.int32)
    if case["kind"] == "compact":          # every second sequence is gone; what is left has a fork that shares its full pages
        table[1:n:2], seq_lens[1:n:2] = -1, 0
        full = seq_lens[0:n:2] // page
        for i, f in enumerate(full):
            table[n + i, :f] = table[2 * i, :f]
            seq_lens[n + i] = f * page
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    books = torch.from_numpy(np.concatenate((table.ravel(), seq_lens, refs))).cuda()
    now = torch.empty_like(books)
    cut = (table.size, table.size + seq_lens.size)
    shape = (case["layers"], pages, kv, page, d)
    state = {"books": books, "now": now, "page_table": now[:cut[0]].view(table.shape), "seq_lens": now[cut[0]:cut[1]],
             "page_refs": now[cut[1]:], "k": torch.randn(shape, generator=gen, device="cuda", dtype=dtype),
             "v": torch.randn(shape, generator=gen, device="cuda", dtype=dtype)}
    if case["kind"] == "branch":
        src = np.random.default_rng(seed).permutation(n).astype(np.int32)
        state["src"] = torch.from_numpy(src).cuda()
        state["dst"] = torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")
        state["counts"] = torch.tensor([0] * n + [1 + i % page for i in range(n)], dtype=torch.int32, device="cuda")
        state["gone"] = state["src"][: n // 2].contiguous()
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"decode": _plain_decode, "append": _plain_append, "branch": _plain_branch, "compact": _plain_compact}[
        state["case"]["kind"]](state)


def _run_own(s):
    import stickbreaking_attention_b200 as sb
    case = s["case"]
    if case["kind"] == "decode":
        o, rem = sb.sb_attn_decode(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"],
                                   attend_current=case["attend_current"])
        return {"o": o, "rem": rem}
    if case["kind"] == "append":
        sb.kv_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], s["cu_seqlens"])
        return {"k": s["k_pages"], "v": s["v_pages"]}
    s["now"].copy_(s["books"])       # the tables as they were, so that every pass does the same work
    books = (s["page_table"], s["seq_lens"], s["page_refs"])
    if case["kind"] == "branch":
        sb.kv_fork(s["k"], s["v"], *books, s["src"], s["dst"])
        sb.kv_extend(*books, s["counts"], case["page"])
        sb.kv_free(*books, s["gone"], case["page"])
    else:
        sb.kv_compact(s["k"], s["v"], *books)
    return _pages_out(s)


def _pages_out(s):
    return {"k": s["k"], "v": s["v"], "page_table": s["page_table"], "seq_lens": s["seq_lens"], "page_refs": s["page_refs"]}


def _plain_decode(s):
    case, q, lens = s["case"], s["q"], s["seq_lens"]
    seqs, heads, new, d = q.shape
    kv = case["kv_heads"]
    at = s["page_table"].clamp(min=0).long()

    def keys(pages):         # (seqs, kv heads, positions, d)
        return pages[at].transpose(1, 2).flatten(2, 3).float()

    k, v = keys(s["k_pages"]), keys(s["v_pages"])
    pos = torch.arange(k.shape[2], device=q.device)
    limit = lens[:, None] - new + torch.arange(new, device=q.device)[None] + int(case["attend_current"])     # (seqs, new)
    allowed = (pos[None, None] < limit[:, :, None])[:, None, None]                              # (seqs, 1, 1, new, positions)
    z = q.view(seqs, kv, heads // kv * new, d).float() @ k.transpose(2, 3) / math.sqrt(d)
    z = z.view(seqs, kv, heads // kv, new, -1)
    # log(1 - beta) = -(max(z, 0) + log1p(exp(-|z|))); over up to 131072 keys its sums are kept in 64 bits
    broken = torch.where(allowed, torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())), 0.0)
    later = broken.double().flip(-1).cumsum(-1).flip(-1)
    a = torch.where(allowed, torch.exp(z - later.float()), 0.0)            # log beta - (what the later keys broke off)
    o = a.view(seqs, kv, heads // kv * new, -1) @ v
    rem = torch.exp(-later[..., 0]).float()
    return {"o": o.view(seqs, heads, new, d).to(q.dtype), "rem": rem.view(seqs, heads, new).to(q.dtype)}


def _plain_append(s):
    case, lens = s["case"], s["seq_lens"].long()
    k, v = s["k"], s["v"]
    if s["cu_seqlens"] is None:
        k, v = k.squeeze(2), v.squeeze(2)                                                  # (seqs, kv heads, d)
        seq = torch.arange(lens.numel(), device=k.device)
        pos = lens - 1
    else:
        k, v = k.transpose(0, 1), v.transpose(0, 1)                                        # (tokens, kv heads, d)
        token = torch.arange(k.shape[0], device=k.device)
        seq = torch.searchsorted(s["cu_seqlens"][1:].long(), token, right=True)
        pos = lens[seq] - s["cu_seqlens"][1:].long()[seq] + token
    at = s["page_table"][seq, pos // case["page"]].long()
    s["k_pages"][at, :, pos % case["page"]] = k
    s["v_pages"][at, :, pos % case["page"]] = v
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_branch(s):
    page = s["case"]["page"]
    s["now"].copy_(s["books"])
    table, lens, refs = s["page_table"], s["seq_lens"], s["page_refs"]
    src, dst = s["src"].long(), s["dst"].long()
    column = torch.arange(table.shape[1], device=table.device)[None]

    # fork: full pages are shared, the rows in use of a last page that is not full are copied to the lowest free pages
    full, rest = (lens[src] // page).long(), lens[src] % page
    part = rest > 0
    free = (refs == 0).nonzero()[:, 0]
    old = table[src[part], full[part]].long()
    new = free[: old.numel()]
    filled = (torch.arange(page, device=table.device)[None] < rest[part][:, None])[None, :, None, :, None]
    for cache in (s["k"], s["v"]):
        cache[:, new] = torch.where(filled, cache[:, old], cache[:, new])
    shared = torch.where(column < full[:, None], table[src], -1)
    table[dst] = shared
    table[dst[part], full[part]] = new.int()
    refs.index_add_(0, shared[shared >= 0].long(), torch.ones_like(shared[shared >= 0]))
    refs[new] = 1
    lens[dst] = lens[src]

    # extend: room for new tokens from the lowest free pages, sequence by sequence
    more = lens + s["counts"]
    fresh = (column >= ((lens + page - 1) // page)[:, None]) & (column < ((more + page - 1) // page)[:, None])
    free = (refs == 0).nonzero()[:, 0][: int(fresh.sum())]
    table[fresh] = free.int()
    refs[free] = 1
    lens.copy_(more)

    # free: the counts go down, the slots are empty
    gone = s["gone"].long()
    held = table[gone]
    refs.index_add_(0, held[held >= 0].long(), -torch.ones_like(held[held >= 0]))
    table[gone] = -1
    lens[gone] = 0
    return _pages_out(s)


def _plain_compact(s):
    s["now"].copy_(s["books"])
    table, refs = s["page_table"], s["page_refs"]
    live = refs > 0
    count = int(live.sum())
    holes = (~live[:count]).nonzero()[:, 0]
    moved = live[count:].nonzero()[:, 0] + count
    s["k"][:, holes] = s["k"][:, moved]
    s["v"][:, holes] = s["v"][:, moved]
    place = torch.arange(refs.numel(), device=refs.device, dtype=torch.int32)
    place[moved] = holes.int()
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], table))
    refs[holes] = refs[moved]
    refs[moved] = 0
    return _pages_out(s)


# ---- what a pass cannot do without, and what it computes ----------------------------------------------------------------

def work(case):
    """Bytes: inputs once, outputs once.  Operations: the two products over the (query, key) pairs whose weight is not exactly 0
    in 32 bits."""
    e, d, kv, lens = ESIZE[case["dtype"]], case["head_dim"], case["kv_heads"], lengths(case)
    if case["kind"] == "decode":
        local = {"spread": 0, "local": kv, "mixed": kv // 2}[case["data"]]
        pairs = sum(n * (kv - local) + min(n, LOCAL_REACH) * local for n in lens)
        rows = case["seqs"] * case["heads"] * case["new"]
        table = 4 * (sum(_page_count(lens, case["page"])) + len(lens))
        return {"bytes": float(2 * pairs * d * e + 2 * rows * d * e + rows * e + table),
                "flops": 4.0 * pairs * case["heads"] // kv * case["new"] * d}
    if case["kind"] == "append":
        tokens = sum(lens) if case["prompts"] else len(lens)
        pages = sum(_page_count(lens, case["page"])) if case["prompts"] else len(lens)
        return {"bytes": float(4 * tokens * kv * d * e + 4 * (pages + len(lens))), "flops": 0.0}
    page, n = case["page"], case["seqs"]
    row = 4 * case["layers"] * kv * d * e                  # K and V, read and written
    counts = _page_count(lens, page)
    books = 4 * (2 * sum(counts) + 4 * n + 2 * (sum(counts) + 3 * n + 5))
    if case["kind"] == "branch":
        return {"bytes": float(row * sum(x % page for x in lens) + books), "flops": 0.0}
    live = sum(counts[::2])                                # of a pool whose live pages lie anywhere, the share behind the front
    pages = sum(counts) + 3 * n + 5
    return {"bytes": float(row * page * live * (1 - live / pages) + books), "flops": 0.0}


def exact(case, seed):
    """Decode: each sequence and head in 64 bits, the stick kept as a running product.  (What is left of it where every head is
    local is below the smallest numbers of the outputs' types.)  The other operators copy and count."""
    if case["kind"] != "decode":
        return None
    s = prepare(case, seed)
    q, heads, kv, new = s["q"], case["heads"], case["kv_heads"], case["new"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    rem = torch.ones(q.shape[:3], dtype=torch.float64, device=q.device)
    group = heads // kv
    for b, n in enumerate(lengths(case)):
        at = s["page_table"][b, : -(-n // case["page"])].long()
        for g in range(kv):
            k = s["k_pages"][at, g].flatten(0, 1)[:n].double()
            v = s["v_pages"][at, g].flatten(0, 1)[:n].double()
            for t in range(new):
                last = n - new + t + int(case["attend_current"])
                if last <= 0:
                    continue
                z = (q[b, g * group:(g + 1) * group, t].double() @ k[:last].T) * case["head_dim"] ** -0.5
                stick = torch.cumprod(torch.sigmoid(-z).flip(1), 1)           # what is left after each key, newest first
                before = torch.cat((torch.ones_like(stick[:, :1]), stick[:, :-1]), 1)
                o[b, g * group:(g + 1) * group, t] = (torch.sigmoid(z).flip(1) * before).flip(1) @ v[:last]
                rem[b, g * group:(g + 1) * group, t] = stick[:, -1]
    return {"o": o, "rem": None if case["data"] == "local" else rem}
