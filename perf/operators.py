"""The work around a decode step that stays on the GPU between two steps: what a server with paged caches, and with beams, has
the framework do from one step's logits to the next step's launch.

    tables    step tables from request lengths: positions, state rows, cache destinations, block tables, window entries, and the
              pages that growing requests take from the free stacks
    select    the next beams: log-softmax over the vocabulary, cumulative scores, the best k over beams x vocabulary
    reorder   the caches of beams that fork: state rings, window ring, the compressed records behind the shared prompt

All inputs are made on the GPU from the seed.  With `own` the calls are this package's; otherwise elementary torch operations.
"""
import numpy as np
import torch

own = False

RATIO, RING, WINDOW, TOPK = 4, 8, 128, 2048      # tokens per compressed entry, state ring, sliding window, selected entries
EPB, SWA_EPB = 64, 256                           # entries per page: compressed pools, window pool
MAIN, INDEX = 2048, 512                          # fp32 values per entry of the two state rings


def listed():
    return [
        # one user's token at a short context: nothing but latency
        dict(name="tables_b1_ctx4096", kind="tables", rows=1, spare=0, lo=4095, hi=4095, budget=0, width=17, padded=0, short=False),
        # the headline decode batch: 64 requests at 32 K tokens, tables as wide as their longest context
        dict(name="tables_b64_ctx32768", kind="tables", rows=64, spare=0, lo=16384, hi=32767, budget=0, width=129, padded=0,
             short=False),
        # the largest decode batch at very long contexts, a few padded rows as a captured batch has them
        dict(name="tables_b128_ctx1m", kind="tables", rows=128, spare=32, lo=65536, hi=1048575, budget=0, width=4097, padded=5,
             short=False),
        # prompts read in chunks of ragged lengths beside decoding requests, the pool running out behind them
        dict(name="tables_b37_chunks", kind="tables", rows=37, spare=11, lo=0, hi=50003, budget=65521, width=256, padded=2,
             short=True),
        # one prompt's beams: four of them, eight candidates
        dict(name="select_g1_w4", kind="select", groups=1, width=4, vocab=32000, k=8, type="bf16", pad=0, finished=0, masked=0),
        # fp32 logits as a head in full precision gives them
        dict(name="select_g16_w4_fp32", kind="select", groups=16, width=4, vocab=131072, k=4, type="fp32", pad=0, finished=0, masked=0),
        # an odd vocabulary in rows of an odd stride, masked tokens (lowest value, -inf, NaN), a finished beam in every group
        dict(name="select_g7_w5_odd", kind="select", groups=7, width=5, vocab=100003, k=10, type="fp16", pad=6, finished=1, masked=64),
        # a full batch: 512 beams over a large vocabulary
        dict(name="select_g64_w8", kind="select", groups=64, width=8, vocab=131072, k=16, type="bf16", pad=0, finished=0, masked=0),
        # four beams a few tokens behind a prompt, two of them replaced
        dict(name="reorder_g1_w4", kind="reorder", groups=1, width=4, prompt=4001, generated=27, forks=2, fp4=False, history=513),
        # sixteen prompts of eight beams, half of the beams replaced, some hundred tokens generated
        dict(name="reorder_g16_w8", kind="reorder", groups=16, width=8, prompt=4096, generated=500, forks=4, fp4=False, history=1024),
        # wide beams far behind their prompts, MXFP4 index records
        dict(name="reorder_g8_w32_fp4", kind="reorder", groups=8, width=32, prompt=10007, generated=2045, forks=20, fp4=True, history=2111),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("tables", "select", "reorder"))
    if kind == "tables":
        rows = _log_int(rng, 1, 512)
        hi = _log_int(rng, 1, min(1048575, 128 * 1048576 // rows))
        chunks = rng.random() < 0.4
        budget = _log_int(rng, rows, 65536) if chunks else 0
        return dict(kind=kind, rows=rows, spare=rng.randrange(0, 40), lo=hi // rng.choice((1, 2, 16)) if rng.random() < 0.8 else 0, hi=hi,
                    budget=budget, width=(hi + min(budget, 8192)) // (RATIO * EPB) + rng.choice((1, 2, 7)),
                    padded=rng.randrange(0, 1 + rows // 8), short=chunks and rng.random() < 0.3)
    if kind == "select":
        width = rng.choice((1, 2, 3, 4, 4, 5, 6, 8, 8, 12, 16, 31, 32))
        vocab = _log_int(rng, 1000, 262144)
        groups = _log_int(rng, 1, max(1, min(128, 64 * 8 * 131072 // (width * vocab))))
        kind_of = rng.choice(("bf16", "fp16", "fp32"))
        if kind_of == "fp32":
            groups = max(1, groups // 2)
        return dict(kind=kind, groups=groups, width=width, vocab=vocab, k=min(64, max(1, width * rng.choice((1, 2)))), type=kind_of,
                    pad=rng.choice((0, 0, 1, 8, 61)), finished=rng.choice((0, 0, min(1, width - 1), width // 2)),
                    masked=rng.choice((0, 0, 64, vocab // 2)))
    width = rng.choice((2, 3, 4, 4, 5, 8, 8, 16, 32))
    groups = _log_int(rng, 1, max(1, 256 // width))
    return dict(kind=kind, groups=groups, width=width, prompt=_log_int(rng, 1, 30000), generated=_log_int(rng, 1, 2000),
                forks=rng.randrange(1, 1 + max(1, width * 5 // 8)), fp4=rng.random() < 0.4, history=_log_int(rng, 16, 2111))


# ---------------------------------------------------------------- what a program holds before the call

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randint(g, lo, hi, *shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)


def _pages_of(tokens):
    return (tokens // RATIO + EPB - 1) // EPB


def _page_tables(g, held, width, spare):
    """Tables [slots, width] over distinct shuffled pages, zero behind what each slot holds, and the pages that are left."""
    first = torch.cumsum(held, 0) - held
    total = int(held.sum())
    shuffled = torch.randperm(total + spare, generator=g, device="cuda").int()
    at = torch.arange(width, device="cuda")[None, :]
    table = torch.where(at < held[:, None], shuffled[(first[:, None] + at).clamp_max(max(total + spare - 1, 0))], 0)
    return table.int().contiguous(), shuffled[total:].contiguous()


def _prepare_tables(c, seed):
    g = _generator(seed)
    rows, width = c["rows"], c["width"]
    capacity = rows + c["spare"]
    slots = torch.randperm(capacity, generator=g, device="cuda")[:rows].int()
    lengths = _randint(g, c["lo"], c["hi"] + 1, capacity)
    new = torch.ones(rows, dtype=torch.int32, device="cuda")
    if c["budget"]:               # a step's tokens cut into one ragged chunk per request
        cuts = torch.cat([_randint(g, 0, c["budget"] + 1, rows - 1).sort().values, new.new_full((1,), c["budget"])])
        new = torch.diff(cuts, prepend=new.new_zeros(1))
    if c["padded"]:
        slots[torch.randperm(rows, generator=g, device="cuda")[:c["padded"]]] = -1
    used = slots.clamp_min(0).long()
    need = torch.where(slots >= 0, _pages_of(lengths[used] + new) - _pages_of(lengths[used]), 0)
    needed = int(need.sum())
    free = max(1, needed * 3 // 4) if c["short"] else needed + 5
    s = dict(kind="tables", slots=slots, lengths=lengths, tokens=c["budget"] or rows, new=new if c["budget"] else None,
             counts=torch.tensor([free, free], dtype=torch.int32, device="cuda"))
    for name in ("idx", "cmp"):
        s[name + "_table"], s[name + "_free"] = _page_tables(g, _pages_of(lengths), width, needed + 5)
    window_pages = -(-WINDOW // SWA_EPB)
    s["swa_table"] = torch.randperm(capacity * window_pages, generator=g, device="cuda").int().view(capacity, window_pages)
    if own:
        import wuda_b200 as wuda
        s["plan"] = wuda.StepTables(s["lengths"], s["idx_table"], s["cmp_table"], s["swa_table"], s["idx_free"], s["cmp_free"], s["counts"],
                                    max_rows=rows, max_tokens=s["tokens"], idx_entries_per_block=EPB, cmp_entries_per_block=EPB,
                                    swa_entries_per_block=SWA_EPB, ratio=RATIO, ring_entries=RING, window=WINDOW, topk=TOPK,
                                    lengths_out=torch.empty_like(lengths), free_counts_out=torch.empty_like(s["counts"]))
    return s


TYPES = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)


def _prepare_select(c, seed):
    g = _generator(seed)
    groups, width, vocab, kind = c["groups"], c["width"], c["vocab"], TYPES[c["type"]]
    held = torch.empty(groups, width, vocab + c["pad"], dtype=kind, device="cuda")
    for at in range(groups):      # a bulk of unlikely tokens, a few likely ones
        part = torch.randn(width, vocab + c["pad"], generator=g, device="cuda") * 2.0
        likely = torch.arange(20, device="cuda") * (vocab // 20) + _randint(g, 0, vocab // 20, width, 20, dtype=torch.int64)
        part.scatter_add_(1, likely, torch.rand(likely.shape, generator=g, device="cuda") * 10)      # (20 different tokens)
        held[at] = part.to(kind)
    logits = held[:, :, :vocab]
    if c["masked"]:
        count = min(c["masked"], vocab - 2 * c["k"])
        for at, value in enumerate((torch.finfo(kind).min, float("-inf"), float("nan"))):
            logits[:, :, torch.randperm(vocab, generator=g, device="cuda")[at:count:3]] = value
    scores = -torch.rand(groups, width, generator=g, device="cuda") * 12 - 20
    finished = None
    if c["finished"]:
        finished = torch.rand(groups, width, generator=g, device="cuda").argsort(1) < c["finished"]
    return dict(kind="select", logits=logits, scores=scores, finished=finished, k=c["k"], eos=2)


def _prepare_reorder(c, seed):
    g = _generator(seed)
    groups, width = c["groups"], c["width"]
    beams = groups * width
    capacity = beams + 3
    length = c["prompt"] + c["generated"]
    slots = torch.randperm(capacity, generator=g, device="cuda")[:beams].int().view(groups, width).contiguous()
    # `forks` beams of each group without a child, their places taken by further children of the others
    order = torch.rand(groups, width, generator=g, device="cuda").argsort(1)
    alive = order[:, :width - c["forks"]]
    extra = torch.gather(alive, 1, _randint(g, 0, alive.size(1), groups, c["forks"], dtype=torch.int64))
    parents = torch.cat([alive, extra], 1)
    parents = torch.gather(parents, 1, torch.rand(groups, width, generator=g, device="cuda").argsort(1)).int().contiguous()
    s = dict(kind="reorder", slots=slots, parents=parents, slots_out=torch.empty_like(slots), records=(64, 4) if c["fp4"] else (128, 4),
             lengths=torch.full((capacity,), length, dtype=torch.int32, device="cuda"),
             shared=torch.full((capacity,), c["prompt"], dtype=torch.int32, device="cuda"))
    s["states"] = [torch.randn(capacity, RING, MAIN, generator=g, device="cuda"), torch.randn(capacity, RING, INDEX, generator=g, device="cuda"),
                   _randint(g, 0, 100000, capacity, c["history"])]
    entries, common = length // RATIO, c["prompt"] // RATIO // EPB
    pages = -(-entries // EPB)
    for name, record in (("idx", sum(s["records"])), ("cmp", 584)):
        # each slot's own pages behind the ones that its group shares
        table = torch.zeros(capacity, pages + 1, dtype=torch.int32, device="cuda")
        perm = torch.randperm(groups * common + capacity * (pages - common), generator=g, device="cuda").int()
        table[:, common:pages] = perm[groups * common:].view(capacity, pages - common)
        table[slots.view(-1).long(), :common] = perm[:groups * common].view(groups, 1, common).expand(groups, width, common).reshape(beams, common)
        s[name + "_table"] = table
        stride = EPB * record if name == "idx" else -(-EPB * record // 576) * 576
        s[name + "_pool"] = _randint(g, 0, 256, max(perm.numel(), 1), stride, dtype=torch.uint8)
    s["swa_table"] = torch.randperm(capacity, generator=g, device="cuda").int().view(capacity, 1)
    s["swa_pool"] = _randint(g, 0, 256, capacity, -(-SWA_EPB * 584 // 576) * 576, dtype=torch.uint8)
    if own:
        import wuda_b200 as wuda
        s["plan"] = wuda.BeamReorder(
            s["lengths"], width, shared_lengths=s["shared"], states=s["states"],
            pools=[wuda.PagedState(s["idx_pool"], s["idx_table"], EPB, s["records"], tokens_per_entry=RATIO),
                   wuda.PagedState(s["cmp_pool"], s["cmp_table"], EPB, (576, 8), tokens_per_entry=RATIO),
                   wuda.PagedState(s["swa_pool"], s["swa_table"], SWA_EPB, (576, 8), ring=WINDOW)])
    return s


def prepare(case, seed):
    return dict(tables=_prepare_tables, select=_prepare_select, reorder=_prepare_reorder)[case["kind"]](case, seed)


# ---------------------------------------------------------------- one pass

TABLE_OUTPUTS = ("pos", "q_pos", "state_row", "idx_dst", "cmp_dst", "swa_dst", "token_starts", "n_compressed", "cmp_lengths",
                 "swa_lengths", "swa_indices", "idx_block_table", "cmp_block_table")


def _run_tables(s):
    if own:
        out = s["plan"].step(s["slots"], s["new"])
        return [out[name] for name in TABLE_OUTPUTS] + [s["plan"].lengths_out, s["plan"].free_counts_out, s["idx_table"], s["cmp_table"]]
    slots, lengths, width = s["slots"].long(), s["lengths"].long(), s["idx_table"].size(1)
    rows, capacity = slots.numel(), lengths.numel()
    dev = slots.device
    new = torch.ones_like(slots) if s["new"] is None else s["new"].long()
    row = torch.arange(rows, device=dev)
    good = (slots >= 0) & (slots < capacity)
    good &= ~((slots[:, None] == slots[None, :]) & (row[None, :] < row[:, None])).any(1)
    slot = torch.where(good, slots, 0)
    end = torch.cumsum(new, 0)
    start = end - new
    old = lengths[slot]
    now = old + new
    held, wanted = _pages_of(old), _pages_of(now)
    good &= (old >= 0) & (wanted <= width) & (end <= s["tokens"])
    need = torch.where(good, wanted - held, 0)
    taken = torch.cumsum(need, 0)
    good &= (need == 0) | ((taken <= s["counts"][0]) & (taken <= s["counts"][1]))
    need = torch.where(good, need, 0)
    zero = lambda value: torch.where(good, value, 0)
    # rows
    out = {}
    entries = zero(now // RATIO)
    out["token_starts"] = torch.cat([end.new_zeros(1), end]).int()
    out["n_compressed"], out["cmp_lengths"] = entries.int(), entries.clamp_max(TOPK).int()
    valid = zero(now.clamp_max(WINDOW))
    out["swa_lengths"] = valid.int()
    at = torch.arange(WINDOW, device=dev)[None, :]
    ring = (now[:, None] - valid[:, None] + at) % WINDOW
    pages = s["swa_table"].long()[slot]
    out["swa_indices"] = torch.where(at < valid[:, None], torch.gather(pages, 1, ring // SWA_EPB) * SWA_EPB + ring % SWA_EPB, -1).int()
    # tokens
    token = torch.arange(s["tokens"], device=dev)
    of = torch.searchsorted(end, token, right=True)
    pos = old[of] + token - start[of]
    keep, slot_of, now_of = good[of], slot[of], now[of]
    out["pos"] = torch.where(keep, pos, 0)
    out["q_pos"] = out["pos"].int()
    out["state_row"] = torch.where(keep & (pos >= now_of - RING), slot_of * RING + pos % RING, -1)
    turn = pos % WINDOW
    out["swa_dst"] = torch.where(keep & (pos >= now_of - WINDOW), s["swa_table"].long()[slot_of, turn.clamp_min(0) // SWA_EPB] * SWA_EPB
                                 + turn % SWA_EPB, -1)
    entry = (pos + 1) // RATIO - 1
    full = keep & ((pos + 1) % RATIO == 0)
    column = torch.arange(width, device=dev)[None, :]
    for at, name in enumerate(("idx", "cmp")):
        stack, table = s[name + "_free"].long(), s[name + "_table"]
        pop = s["counts"][at].long() - 1 - ((taken - need)[:, None] + column - held[:, None])
        grown = good[:, None] & (column >= held[:, None]) & (column < (held + need)[:, None])
        there = table.long()[slot]
        there = torch.where(grown, stack[pop.clamp(0, stack.numel() - 1)], there)
        block = torch.where(good[:, None] & (column < wanted[:, None]), there, 0)
        out[name + "_block_table"] = block.int()
        where = torch.where(full, entry, 0)
        out[name + "_dst"] = torch.where(full, block[of, where // EPB] * EPB + where % EPB, -1)
        spread = grown.nonzero(as_tuple=True)
        table[slot[spread[0]], spread[1]] = block[spread].int()
    after = s["lengths"].clone()
    after[slots[good]] = now[good].int()
    counts = (s["counts"] - need.sum()).int()
    return [out[name] for name in TABLE_OUTPUTS] + [after, counts, s["idx_table"], s["cmp_table"]]


def _run_select(s):
    if own:
        import wuda_b200 as wuda
        return wuda.beam_select(s["logits"], s["scores"], s["k"], finished=s["finished"], eos_token=s["eos"])
    logits, scores, k, eos = s["logits"], s["scores"], s["k"], s["eos"]
    groups, width, vocab = logits.shape
    x = logits.float()
    x = torch.where(torch.isfinite(x), x, float("-inf"))
    top = x.amax(2, keepdim=True)
    total = torch.exp(x - top).sum(2, dtype=torch.float64)
    lse = top.squeeze(2).double() + total.log()
    # the best k of every beam, ties to the lower token: unique keys of (value, token)
    bits = x.contiguous().view(torch.int32).long()
    bits = torch.where(bits < 0, torch.bitwise_xor(bits, 0x7fffffff), bits)
    keys = (bits << 32) | (0xffffffff - torch.arange(vocab, device=x.device))
    token = 0xffffffff - (torch.topk(keys, min(k, vocab), dim=2).values & 0xffffffff)
    best = torch.gather(x, 2, token).double()
    value = scores.double()[:, :, None] + (best - lse[:, :, None])
    if s["finished"] is not None:
        alone = torch.full_like(value, float("-inf"))
        alone[:, :, 0] = scores.double()
        value = torch.where(s["finished"][:, :, None], alone, value)
        token = torch.where(s["finished"][:, :, None], eos, token)
    value, order = torch.sort(value.view(groups, -1), dim=1, descending=True, stable=True)
    order, value = order[:, :k], value[:, :k]
    parents = order // token.size(2)
    tokens = torch.gather(token.view(groups, -1), 1, order)
    done = tokens == eos
    if s["finished"] is not None:
        done |= torch.gather(s["finished"], 1, parents)
    return value.float(), parents.int(), tokens.int(), done


def _forks(parents, slots):
    """New slots, and source and destination slot of every fork."""
    groups, width = parents.shape
    parents = parents.long()
    beam = torch.arange(width, device=parents.device)
    older = (parents[:, None, :] == parents[:, :, None]) & (beam[None, None, :] < beam[None, :, None])
    extra = older.any(2)                                            # another child of a parent that keeps its slot
    childless = ~(parents[:, None, :] == beam[None, :, None]).any(2)
    source = torch.gather(slots, 1, parents)
    places = torch.argsort((~childless).long(), dim=1, stable=True)                   # childless beams first, in their order
    rank = (torch.cumsum(extra.long(), 1) - 1).clamp_min(0)
    out = torch.where(extra, torch.gather(slots, 1, torch.gather(places, 1, rank)), source)
    return out, source[extra].long(), out[extra].long()


def _run_reorder(s):
    if own:
        s["plan"].run(s["parents"], s["slots"], s["slots_out"])
        return [s["slots_out"]] + s["states"] + [s["idx_pool"], s["cmp_pool"], s["swa_pool"]]
    out, src, dst = _forks(s["parents"], s["slots"])
    for state in s["states"]:
        state[dst] = state[src]
    length, shared = s["lengths"].long()[src], s["shared"].long()[src]
    for name, epb, parts in (("idx", EPB, s["records"]), ("cmp", EPB, (576, 8)), ("swa", SWA_EPB, (576, 8))):
        pool, table = s[name + "_pool"], s[name + "_table"].long()
        width = table.size(1)
        entries = length.clamp_max(WINDOW) if name == "swa" else length // RATIO
        first = torch.zeros_like(entries) if name == "swa" else shared // RATIO // epb * epb
        at = torch.arange(width * epb, device=pool.device)[None, :]
        fork, entry = ((at >= first[:, None]) & (at < entries[:, None])).nonzero(as_tuple=True)
        from_page, to_page = table[src[fork], entry // epb], table[dst[fork], entry // epb]
        offset = 0
        for size in parts:
            view = pool[:, offset:offset + epb * size].unflatten(1, (epb, size))
            view[to_page, entry % epb] = view[from_page, entry % epb]
            offset += epb * size
    return [out] + s["states"] + [s["idx_pool"], s["cmp_pool"], s["swa_pool"]]


def run(state):
    return dict(tables=_run_tables, select=_run_select, reorder=_run_reorder)[state["kind"]](state)


# ---------------------------------------------------------------- the same from the definitions, row by row and in 64 bits

def _exact_tables(s):
    a = {k: v.cpu().numpy().astype(np.int64) for k, v in s.items() if isinstance(v, torch.Tensor)}
    slots, lengths, width = a["slots"], a["lengths"].copy(), a["idx_table"].shape[1]
    rows, tokens = len(slots), s["tokens"]
    new = np.ones(rows, np.int64) if s["new"] is None else a["new"]
    out = {n: np.zeros(tokens, np.int64) for n in ("pos", "state_row", "idx_dst", "cmp_dst", "swa_dst")}
    out.update({n: np.zeros(rows, np.int64) for n in ("n_compressed", "cmp_lengths", "swa_lengths")},
               swa_indices=np.full((rows, WINDOW), -1, np.int64), idx_block_table=np.zeros((rows, width), np.int64),
               cmp_block_table=np.zeros((rows, width), np.int64), token_starts=np.zeros(rows + 1, np.int64))
    for name in ("state_row", "idx_dst", "cmp_dst", "swa_dst"):
        out[name][:] = -1
    free = {n: a[n + "_free"][:a["counts"][i]].tolist() for i, n in enumerate(("idx", "cmp"))}
    seen, stopped, at = set(), False, 0
    for b in range(rows):
        slot, n = int(slots[b]), int(new[b])
        t0, at = at, at + n
        out["token_starts"][b + 1] = at
        if not 0 <= slot < len(lengths) or slot in seen:
            continue
        seen.add(slot)
        old = int(lengths[slot])
        now = old + n
        need = -(-(now // RATIO) // EPB) - -(-(old // RATIO) // EPB)
        if old < 0 or -(-(now // RATIO) // EPB) > width or at > tokens:
            continue
        if need and (stopped or need > len(free["idx"]) or need > len(free["cmp"])):
            stopped = True
            continue
        lengths[slot] = now
        p = np.arange(old, now)
        out["pos"][t0:at] = p
        out["state_row"][t0:at] = np.where(p >= now - RING, slot * RING + p % RING, -1)
        ring = p % WINDOW
        out["swa_dst"][t0:at] = np.where(p >= now - WINDOW, a["swa_table"][slot, ring // SWA_EPB] * SWA_EPB + ring % SWA_EPB, -1)
        out["n_compressed"][b], out["cmp_lengths"][b] = now // RATIO, min(now // RATIO, TOPK)
        last = np.arange(max(0, now - WINDOW), now) % WINDOW
        out["swa_lengths"][b] = len(last)
        out["swa_indices"][b, :len(last)] = a["swa_table"][slot, last // SWA_EPB] * SWA_EPB + last % SWA_EPB
        for name in ("idx", "cmp"):
            table = a[name + "_table"][slot]
            held = -(-(old // RATIO) // EPB)
            for page in range(held, held + need):
                table[page] = free[name].pop()
            out[name + "_block_table"][b, :held + need] = table[:held + need]
            e = (p + 1) // RATIO - 1
            out[name + "_dst"][t0:at] = np.where((p + 1) % RATIO == 0, table[np.maximum(e, 0) // EPB] * EPB + e % EPB, -1)
    out["q_pos"] = out["pos"]
    wide = ("pos", "state_row", "idx_dst", "cmp_dst", "swa_dst")
    result = [torch.from_numpy(out[n] if n in wide else out[n].astype(np.int32)).cuda() for n in TABLE_OUTPUTS]
    counts = np.array([len(free["idx"]), len(free["cmp"])])
    return result + [torch.from_numpy(v.astype(np.int32)).cuda() for v in (lengths, counts, a["idx_table"], a["cmp_table"])]


def _exact_select(s):
    groups, width, vocab = s["logits"].shape
    values, parents, tokens, done = [], [], [], []
    for at in range(groups):
        x = s["logits"][at].double()
        x = x.masked_fill(~(x.abs() < float("inf")), float("-inf"))
        value = s["scores"][at].double()[:, None] + torch.log_softmax(x, 1)
        ended = torch.zeros(width, dtype=torch.bool, device=x.device) if s["finished"] is None else s["finished"][at]
        value[ended] = float("-inf")
        value[ended, s["eos"]] = s["scores"][at].double()[ended]
        best, order = torch.sort(value.view(-1), descending=True, stable=True)
        best, order = best[:s["k"]], order[:s["k"]]
        values.append(best)
        parents.append((order // vocab).int())
        tokens.append((order % vocab).int())
        done.append((order % vocab == s["eos"]) | ended[order // vocab])
    return tuple(torch.stack(v) for v in (values, parents, tokens, done))


def _exact_reorder(s):
    parents, slots = s["parents"].cpu().numpy(), s["slots"].cpu().numpy()
    out = slots.copy()
    moves = []
    for p, now, new in zip(parents, slots, out):
        unused = [beam for beam in range(len(p)) if beam not in p]
        seen = set()
        for beam, parent in enumerate(p.tolist()):
            if parent in seen:
                new[beam] = now[unused.pop(0)]
                moves.append((int(now[parent]), int(new[beam])))
            else:
                new[beam] = now[parent]
            seen.add(parent)
    length, shared = int(s["lengths"][0]), int(s["shared"][0])
    states = [t.clone() for t in s["states"]]
    pools = []
    for name, epb, parts in (("idx", EPB, s["records"]), ("cmp", EPB, (576, 8)), ("swa", SWA_EPB, (576, 8))):
        pool, table = s[name + "_pool"].clone(), s[name + "_table"].cpu().numpy()
        entries, first = (min(length, WINDOW), 0) if name == "swa" else (length // RATIO, shared // RATIO // epb)
        for src, dst in moves:
            for page in range(first, -(-entries // epb)):
                count, offset = min(epb, entries - page * epb), 0
                for size in parts:
                    pool[int(table[dst, page]), offset:offset + count * size] = pool[int(table[src, page]), offset:offset + count * size]
                    offset += epb * size
        pools.append(pool)
    for state in states:
        for src, dst in moves:
            state[dst].copy_(state[src])
    return [torch.from_numpy(out).to(s["slots"].device)] + states + pools


def exact(case, seed):
    s = prepare(case, seed)
    return dict(tables=_exact_tables, select=_exact_select, reorder=_exact_reorder)[case["kind"]](s)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "tables":
        rows = c["rows"]
        tokens = c["budget"] or rows
        pages = (c["lo"] + c["hi"]) / 2 / (RATIO * EPB)
        # slots, lengths and pages held are read; tokens, row values, window entries and the whole tables are written
        moved = rows * 12 + rows * pages * 2 * 4 + tokens * (5 * 8 + 4) + rows * (4 * 4 + WINDOW * 4) + rows * c["width"] * 2 * 4
        return dict(bytes=moved, flops=tokens * 12 + rows * c["width"] * 2)
    if c["kind"] == "select":
        size = 4 if c["type"] == "fp32" else 2
        beams = c["groups"] * (c["width"] - c["finished"])
        return dict(bytes=beams * c["vocab"] * size + c["groups"] * (c["width"] * 5 + c["k"] * 13), flops=beams * c["vocab"] * 4)
    length = c["prompt"] + c["generated"]
    entries = length // RATIO - c["prompt"] // RATIO // EPB * EPB
    moved = RING * (MAIN + INDEX) * 4 + c["history"] * 4 + min(length, WINDOW) * 584 + entries * ((68 if c["fp4"] else 132) + 584)
    return dict(bytes=2 * c["groups"] * c["forks"] * moved + c["groups"] * c["width"] * 12, flops=0)
