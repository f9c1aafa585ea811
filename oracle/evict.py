"""float64 numpy definition of the scored and differential decode, the append and the eviction
of a paged cache. TEST INFRASTRUCTURE ONLY (no reference counterpart).

Each attention function also returns how far an fp32 computation may be off, derived from the
arithmetic and not from a run:

  * a logit is a sum of D products on the tensor core. The products of two 16-bit numbers are exact;
    each of the D / 16 accumulation steps may truncate 17 terms at 2^-23 of the largest, and the
    scale is one more product: |dx| <= (D / 16 + 3) * 2^-21 * scale * sum |q_i k_i|.
  * a weight is 2^(x - m) / L: relative error |dx| (numerator) + |dx| (sum) + 16 roundings of 2^-23
    (two exponentials of 2 ulp each, the joins of warps and splits, the quotient) + the precision
    of a weight on its way to the values: 2^-21 for fp16 pairs (or 2^-40 of the largest weight,
    where that is more: `tests/test_evict_weights_gpu.py`); the three bf16 limbs are exact, and
    2^-16, which a pair of them would have, is a bound with room.
  * a value product then adds at most its weights' errors times |v|, and fp32 sums of the
    partial products: one tile per 16 tokens, joined pairwise by warps and splits; the running
    sum of n / 32 tiles rounds at 2^-24 of its magnitude each time, in a random walk:
    sqrt(n) * 2^-23 of sum p |v| covers it with room.
"""
import numpy as np


def slots_of(cache, row, n):
    """Rows [n, heads, D] of one sequence in float64."""
    bs = cache.shape[1]
    t = np.arange(n)
    return cache[row[t // bs], t % bs].astype(np.float64)


def _weights(q, k, scale):
    """Softmax weights [n] and the relative error that an fp32 computation may give them."""
    D = q.shape[0]
    x = k @ q * scale
    dx = (D / 16 + 3) * 2.0 ** -21 * scale * (np.abs(k) @ np.abs(q))
    e = np.exp(x - x.max())
    return e / e.sum(), float(2 * dx.max() + 16 * 2.0 ** -23)


def decode(q, k_cache, v_cache, block_table, seq_lens, lam=None, norm_weight=None, norm_eps=1e-5,
           out_scale=1.0, scale=None, pair_bits=21):
    """-> out [B, H, width], its fp32 error bound, and per sequence the weight that
    each token adds to its score [Hkv, n] with that bound. lam [B, H] selects the differential
    form. q and the caches are arrays of any float type that numpy can widen."""
    B, Hq, D = q.shape
    maps = 1 if lam is None else 2
    Hkv = v_cache.shape[2]
    H = Hq // maps
    G = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = np.zeros((B, H, v_cache.shape[3]))
    tol = np.zeros_like(out)
    added = []
    for b in range(B):
        n = int(seq_lens[b])
        k, v = slots_of(k_cache, block_table[b], n), slots_of(v_cache, block_table[b], n)
        add, add_tol = np.zeros((Hkv, n)), np.zeros((Hkv, n))
        for j in range(H if n else 0):
            h = j // G
            a, ea = _weights(q[b, maps * j].astype(np.float64), k[:, maps * h], scale)
            err = ea * a
            mag = a
            if maps == 2:
                a2, e2 = _weights(q[b, 2 * j + 1].astype(np.float64), k[:, 2 * h + 1], scale)
                lj = float(lam[b, j])
                err = err + abs(lj) * (e2 + 2.0 ** -23) * a2
                mag = a + abs(lj) * a2
                a = a - lj * a2
            add[h] += np.abs(a)
            add_tol[h] += err + 2.0 ** -23 * mag * 2
            o = a @ v[:, h]
            eo = (err + (2.0 ** -pair_bits + np.sqrt(n) * 2.0 ** -23) * mag) @ np.abs(v[:, h])
            if norm_weight is not None:
                r = 1.0 / np.sqrt((o * o).mean() + norm_eps)
                w = norm_weight.astype(np.float64)
                eo = np.abs(w) * r * (eo + np.abs(o) * (r * np.sqrt((eo * eo).mean()) +
                                                        8 * 2.0 ** -23))
                o = o * r * w
            out[b, j] = out_scale * o
            tol[b, j] = abs(out_scale) * eo + 2.0 ** -22 * np.abs(out[b, j])
        added.append((add, add_tol))
    return out, tol, added


def select(scores, positions, seq_lens, next_pos, budget, recent=0, sinks=0):
    """-> src, dst [B, H, M], counts [B, H], new_lens [B], slot by slot."""
    B, H, T = scores.shape
    M = max(1, min(budget, T - budget))
    src = np.full((B, H, M), -1, np.int32)
    dst = np.full((B, H, M), -1, np.int32)
    counts = np.zeros((B, H), np.int32)
    new = np.zeros(B, np.int32)
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), T)
        new[b] = min(n, budget)
        if n <= budget:
            continue
        for h in range(H):
            def rank(t):
                p, s = int(positions[b, h, t]), float(scores[b, h, t])
                if p < sinks or p >= int(next_pos[b]) - recent:
                    return (0, 0.0, t)
                return (2, 0.0, t) if s != s else (1, -s, t)
            kept = set(sorted(range(n), key=rank)[:budget])
            holes = [t for t in range(budget) if t not in kept]
            movers = sorted((t for t in kept if t >= budget), reverse=True)
            counts[b, h] = len(movers)
            src[b, h, :len(movers)] = movers
            dst[b, h, :len(movers)] = holes
    return src, dst, counts, new


def compact(cache, block_table, src, dst, counts):
    """The moves on one paged cache [num_blocks, block_size, H, D] -> a new array."""
    out, bs = cache.copy(), cache.shape[1]
    for b in range(src.shape[0]):
        for h in range(src.shape[1]):
            for i in range(int(counts[b, h])):
                f, t = int(src[b, h, i]), int(dst[b, h, i])
                out[block_table[b, t // bs], t % bs, h] = cache[block_table[b, f // bs], f % bs, h]
    return out


def compact_rows(rows, src, dst, counts):
    """The moves on scores or positions [B, H, T] -> a new array."""
    out = rows.copy()
    for b in range(src.shape[0]):
        for h in range(src.shape[1]):
            for i in range(int(counts[b, h])):
                out[b, h, dst[b, h, i]] = rows[b, h, src[b, h, i]]
    return out


def append(cache, new, new_lens, seq_lens, block_table):
    """Tokens t < new_lens[b] of new [B, S, H, D] to slots seq_lens[b] + t -> a new array."""
    out, bs = cache.copy(), cache.shape[1]
    for b in range(new.shape[0]):
        for t in range(min(int(new_lens[b]), new.shape[1])):
            s = int(seq_lens[b]) + t
            if 0 <= s < block_table.shape[1] * bs:
                out[block_table[b, s // bs], s % bs] = new[b, t]
    return out
