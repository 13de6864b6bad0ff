"""Plain 64-bit implementations of the speculative-decoding operators (step
tables, key bounds, choice of blocks, attention over chosen blocks, draft
verification), written from their definitions with loops over rows.  Only the
tests use them."""
import math

import numpy as np


def step_tables(seq, new, tables, have, free, count, bs, num_blocks, max_tokens):
    """The step's arrays as a dict of int64 numpy arrays, and its status."""
    n, width = tables.shape
    bad = not 0 <= count <= len(free) or sum(int(x) for x in new) > max_tokens
    for i in range(n):
        if seq[i] < 0 or new[i] < 0 or not 0 <= have[i] <= width \
                or -(-(int(seq[i]) + int(new[i])) // bs) > width:
            bad = True
    need = [0] * n
    if not bad:
        need = [max(0, -(-(int(seq[i]) + int(new[i])) // bs) - int(have[i])) for i in range(n)]
    status = -1 if bad else max(0, sum(need) - count)
    ok = status == 0
    left = list(free[:count]) if 0 <= count <= len(free) else []
    out = np.zeros_like(tables)
    pos, slot, cu, blocks = [], [], [0], []
    for i in range(n):
        row = list(tables[i][:min(max(have[i], 0), width)])
        if ok:
            row += [left.pop() for _ in range(need[i])]
            for t in range(int(new[i])):
                p = int(seq[i]) + t
                b = int(row[p // bs])
                pos.append(p)
                slot.append(b * bs + p % bs if 0 <= b < num_blocks else 2 ** 31 - 1)
        out[i, :len(row)] = row
        blocks.append(len(row) if ok else have[i])
        cu.append(len(pos))
    pad = [-1] * (max_tokens - len(pos))
    return {"block_tables": out, "n_blocks": np.array(blocks, np.int64),
            "free_count": np.array([len(left) if ok else count]),
            "context_lens": np.array([s + (m if ok else 0) for s, m in zip(seq, new)], np.int64),
            "cu_q_lens": np.array(cu), "positions": np.array(pos + pad, np.int64),
            "slot_mapping": np.array(slot + pad, np.int64), "status": np.array([status])}


def key_bounds(bounds, k, tables, first, ctx, bs):
    """k: (num_blocks, bs, kv, hd); bounds (num_blocks, kv, 2, hd), updated."""
    for s in range(len(ctx)):
        if ctx[s] <= first[s]:
            continue
        for j in range(first[s] // bs, (ctx[s] - 1) // bs + 1):
            keys = k[tables[s, j], :min(bs, ctx[s] - j * bs)]
            bounds[tables[s, j], :, 0] = keys.min(0)
            bounds[tables[s, j], :, 1] = keys.max(0)
    return bounds


def rows_of(cu, ctx):
    """(sequence, number of keys) of every row; cu None: one row each."""
    if cu is None:
        return [(s, int(c)) for s, c in enumerate(ctx)]
    out = []
    for s, c in enumerate(ctx):
        m = cu[s + 1] - cu[s]
        out += [(s, max(0, int(c) - m + i + 1)) for i in range(m)]
    return out


def block_scores(q, bounds, table, n):
    """(kv, n) float64: max over the group's heads of the bound of q . k in the
    first n blocks of `table`; not finite in the query or the block: +inf."""
    h, hd = q.shape
    b = bounds[table[:n]].astype(np.float64)  # (n, kv, 2, hd)
    kv = b.shape[1]
    with np.errstate(invalid="ignore"):
        x = q.astype(np.float64).reshape(kv, h // kv, 1, hd)
        b = b.transpose(1, 0, 2, 3)[:, None]  # (kv, 1, n, 2, hd)
        s = np.maximum(x * b[..., 0, :], x * b[..., 1, :]).sum(-1)  # (kv, group, n)
        fin = np.isfinite(b).all((-1, -2)) & np.isfinite(x).all(-1)
        s = np.where(fin, s, np.inf)
    return s.max(1)


def select(q, bounds, tables, cu, ctx, bs, top, first, last):
    rows = rows_of(cu, ctx)
    kv = bounds.shape[1]
    out = np.full((len(rows), kv, top), -1, np.int64)
    for r, (s, keys) in enumerate(rows):
        nb = -(-keys // bs)
        if nb <= top:
            out[r, :, :nb] = np.arange(nb)
            continue
        sc = block_scores(q[r], bounds, tables[s], nb)
        for g in range(kv):
            mid = np.arange(first, nb - last)
            best = mid[np.argsort(-sc[g, mid], kind="stable")[:top - first - last]]
            out[r, g] = np.sort(np.concatenate((np.arange(first), best,
                                                np.arange(nb - last, nb))))
    return out


def sparse_attention(q, k, v, blocks, tables, cu, ctx, bs, scale):
    """(out, bound): out (rows, H, hd) in float64; bound: how far a kernel with
    f32 accumulation may be from it.  Score errors: hd + 8 roundings (products,
    sums, scale, the change of base) of the sum of magnitudes; they and two
    exponentials (of a weight and of its rescaling, a few ulp each) change a
    weight's share by twice their size; L additions with the weights."""
    rows = rows_of(cu, ctx)
    h, hd = q.shape[1:]
    kv = k.shape[2]
    out = np.zeros((len(rows), h, hd))
    bound = np.zeros((len(rows), h, 1))
    u = 2.0 ** -24
    for r, (s, keys) in enumerate(rows):
        for g in range(kv):
            pos = [b * bs + o for b in blocks[r, g] if b >= 0 for o in range(bs) if b * bs + o < keys]
            if not pos:
                continue
            pos = np.array(pos)
            blk = tables[s, pos // bs]
            kk, vv = (x[blk, pos % bs, g].astype(np.float64) for x in (k, v))
            for i in range(g * (h // kv), (g + 1) * (h // kv)):
                x = q[r, i].astype(np.float64) @ kk.T * scale
                mag = np.abs(q[r, i]).astype(np.float64) @ np.abs(kk).T * abs(scale)
                e = np.exp(x - x.max())
                out[r, i] = e @ vv / e.sum()
                d = (hd + 8) * u * mag.max() + 16 * u
                bound[r, i] = (2 * d + (len(pos) + 64) * u) * np.abs(vv).max()
    return out, bound


def verify(target, draft_tokens, cu, u, u_last, draft=None, temps=None):
    """(tokens, accepted) with Python lists and float64 sums."""
    batch, vocab = len(cu) - 1, target.shape[1]
    tokens = np.full(target.shape[0], -1, np.int64)
    accepted = np.zeros(batch, np.int64)

    def best(x):
        x = np.where(np.isnan(x), -np.inf, x)
        return int(np.argmax(x)), x.max() > -np.inf

    def dist(x, t):
        x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
        m = x.max()
        if m == -np.inf:
            return np.zeros_like(x)
        with np.errstate(invalid="ignore"):
            w = np.where(x == m, 1.0, np.exp((x - m) / t))
        return w / w.sum()

    for b in range(batch):
        t = 0.0 if temps is None else float(temps[b])
        n, r0 = cu[b + 1] - cu[b], cu[b] + b
        kept = 0
        for i in range(n):
            d = int(draft_tokens[cu[b] + i])
            if not 0 <= d < vocab:
                break
            if t == 0.0:
                top, some = best(target[r0 + i])
                if not some or d != top:
                    break
            else:
                p = dist(target[r0 + i], t)
                q = 1.0 if draft is None else dist(draft[cu[b] + i], t)[d]
                if not float(u[cu[b] + i]) * q < p[d]:
                    break
            kept += 1
        accepted[b] = kept
        tokens[r0:r0 + kept] = draft_tokens[cu[b]:cu[b] + kept]
        if t == 0.0:
            tokens[r0 + kept] = best(target[r0 + kept])[0]
            continue
        p = dist(target[r0 + kept], t)
        w = p
        if kept < n:
            if draft is None:
                w = p.copy()
                d = int(draft_tokens[cu[b] + kept])
                if 0 <= d < vocab:
                    w[d] = 0.0
            else:
                w = np.maximum(p - dist(draft[cu[b] + kept], t), 0.0)
            if not w.sum() > 0:
                w = p
        c = np.cumsum(w)
        hit = np.nonzero((c > float(u_last[b]) * c[-1]) & (w > 0))[0]
        some = np.nonzero(w > 0)[0]
        tokens[r0 + kept] = hit[0] if hit.size else some[-1] if some.size else 0
    return tokens, accepted


def softmax_scale(hd):
    return 1.0 / math.sqrt(hd)
