"""Step tables, beam selection and beam reordering as their definitions say, one row, candidate and entry after the other, in
Python integers and 64-bit floats."""
import numpy as np


def pages_of(tokens, ratio, epb):
    return -(-(tokens // ratio) // epb)


def step_tables(slots, new_tokens, lengths, idx_table, cmp_table, swa_table, idx_free, cmp_free, free_counts, max_tokens, *, idx_epb,
                cmp_epb, swa_epb, ratio, ring, window, topk):
    """All arguments numpy arrays or numbers.  Returns a dict of the outputs and of the state after the step."""
    rows, width = len(slots), idx_table.shape[1]
    new_tokens = np.ones(rows, int) if new_tokens is None else new_tokens
    tables = {"idx": idx_table.copy(), "cmp": cmp_table.copy()}
    stacks = {"idx": idx_free[:free_counts[0]].tolist(), "cmp": cmp_free[:free_counts[1]].tolist()}
    epbs = {"idx": idx_epb, "cmp": cmp_epb}
    lengths = lengths.copy()
    tokens = []          # (pos, state_row, idx_dst, cmp_dst, swa_dst) in order
    rows_out = []        # (n_compressed, swa indices, idx block table, cmp block table)
    starts, seen, stopped, left_out = [0], set(), False, 0
    for slot, n in zip(slots.tolist(), new_tokens.tolist()):
        end = starts[-1] + max(n, 0)
        starts.append(end)
        served = 0 <= slot < len(lengths) and slot not in seen
        if served:
            seen.add(slot)
            old = int(lengths[slot])
            now = old + n
            served = old >= 0 and n >= 0 and now < 2 ** 31 and all(pages_of(now, ratio, e) <= width for e in epbs.values())
        if served:
            need = {p: pages_of(now, ratio, e) - pages_of(old, ratio, e) for p, e in epbs.items()}
            if end > max_tokens:
                stopped, served = True, False
            elif any(need.values()):
                if stopped or any(need[p] > len(stacks[p]) for p in need):
                    stopped, served = True, False
        if not served:
            left_out += slot != -1
            tokens += [(0, -1, -1, -1, -1)] * min(max(n, 0), max_tokens)      # (those beyond the buffers are cut below)
            rows_out.append((0, [], [], []))
            continue
        lengths[slot] = now
        for p, e in epbs.items():
            held = pages_of(old, ratio, e)
            for page in range(held, held + need[p]):
                tables[p][slot, page] = stacks[p].pop()
        place = lambda pages, entry, e: int(pages[entry // e]) * e + entry % e
        for pos in range(old, now):
            entry = (pos + 1) // ratio - 1
            writes = (pos + 1) % ratio == 0
            tokens.append((pos, slot * ring + pos % ring if pos >= now - ring else -1,
                           place(tables["idx"][slot], entry, idx_epb) if writes else -1,
                           place(tables["cmp"][slot], entry, cmp_epb) if writes else -1,
                           place(swa_table[slot], pos % window, swa_epb) if pos >= now - window else -1))
        rows_out.append((now // ratio, [place(swa_table[slot], pos % window, swa_epb) for pos in range(max(0, now - window), now)],
                         tables["idx"][slot, :pages_of(now, ratio, idx_epb)].tolist(), tables["cmp"][slot, :pages_of(now, ratio, cmp_epb)].tolist()))
    tokens = tokens[:max_tokens]
    column = lambda i: np.array([t[i] for t in tokens], np.int64)
    padded = lambda v, n, fill: np.array([x + [fill] * (n - len(x)) for x in v], np.int32).reshape(len(v), n)
    n = np.array([r[0] for r in rows_out], np.int32)
    return dict(pos=column(0), q_pos=column(0).astype(np.int32), state_row=column(1), idx_dst=column(2), cmp_dst=column(3), swa_dst=column(4),
                token_starts=np.minimum(np.array(starts), max_tokens).astype(np.int32), n_compressed=n, cmp_lengths=np.minimum(n, topk),
                swa_lengths=np.array([len(r[1]) for r in rows_out], np.int32), swa_indices=padded([r[1] for r in rows_out], window, -1),
                idx_block_table=padded([r[2] for r in rows_out], width, 0), cmp_block_table=padded([r[3] for r in rows_out], width, 0),
                lengths=lengths, counts=np.array([len(stacks["idx"]), len(stacks["cmp"])], np.int32), idx_table=tables["idx"],
                cmp_table=tables["cmp"], left_out=left_out)


def beam_select(logits, scores, k, finished, eos):
    """logits float64 [groups, width, vocab] of the given values, scores [groups, width].  Returns values (float64), parents,
    tokens, finished, with (-inf, -1, -1, False) behind the last candidate."""
    groups, width, vocab = logits.shape
    values, parents, tokens = np.full((groups, k), -np.inf), np.full((groups, k), -1), np.full((groups, k), -1)
    done = np.zeros((groups, k), bool)
    for g in range(groups):
        found = []
        for w in range(width):
            if not np.isfinite(scores[g, w]):
                continue
            if finished is not None and finished[g, w]:
                found.append((-float(scores[g, w]), w, 0, eos))
                continue
            x = np.where(np.isfinite(logits[g, w]), logits[g, w], -np.inf)
            top = x.max()
            if top == -np.inf:
                continue
            lse = top + np.log(np.exp(x - top).sum())
            order = np.argsort(-x, kind="stable")[:k]
            found += [(-((float(scores[g, w]) + x[v]) - lse), w, i, int(v)) for i, v in enumerate(order) if x[v] > -np.inf]
        for j, (value, w, _, v) in enumerate(sorted(found)[:k]):
            values[g, j], parents[g, j], tokens[g, j] = -value, w, v
            done[g, j] = v == eos or (finished is not None and bool(finished[g, w]))
    return values, parents, tokens, done


def beam_slots(parents, slots, capacity):
    """New slots and (source, destination) of the forks."""
    out, moves = np.full_like(slots, -1), []
    seen = set()
    good = np.zeros(slots.shape, bool)
    for at, s in enumerate(slots.ravel()):
        if 0 <= s < capacity and s not in seen:
            seen.add(int(s))
            good.flat[at] = True
    for g in range(len(parents)):
        width = len(parents[g])
        parent = [int(p) if 0 <= p < width and good[g, p] else -1 for p in parents[g]]
        places = [w for w in range(width) if good[g, w] and w not in parent]
        further, first = [], set()
        for j, p in enumerate(parent):
            if p >= 0 and p not in first:
                first.add(p)
                out[g, j] = slots[g, p]
            elif p >= 0:
                further.append(j)
        for j in further:
            if places:
                out[g, j] = slots[g, places.pop(0)]
                moves.append((g, j, int(slots[g, parent[j]]), int(out[g, j])))
        for j, p in enumerate(parent):
            if p < 0 and places:
                out[g, j] = slots[g, places.pop(0)]
    return out, moves
