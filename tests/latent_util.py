"""Oracles of the latent-cache operators, in 64 bits and on the CPU: an MXFP8 cache in numpy, the attention over a paged
cache, and draft verification."""
import numpy as np

import k3o

PAGE, LATENT, ROPE, ROW, MX8_PAGE = 64, 512, 64, 576, 41984
ROPE_AT, SCALES_AT = 32768, 40960

_E4M3 = np.array([(-1.0 if c & 128 else 1.0) * ((c & 7) / 8 * 2.0 ** -6 if (c >> 3) & 15 == 0 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7))
                  for c in range(256)])
_E4M3[[0x7F, 0xFF]] = np.nan


def quant_rows(rows):
    """[n, 576] bf16 bits -> (codes [n, 512] u8, rope [n, 64] bf16 bits, scales [n, 16] u8); the block quantiser is the
    pinned oracle's."""
    q, sf = k3o.moe_quant(np.ascontiguousarray(rows[:, :LATENT]))
    return q, rows[:, LATENT:], sf


def put_rows(cache, layer_off, page_stride, slots, rows):
    """Append rows to a flat u8 MXFP8 cache, as k3g_latent_mx8_store."""
    q, rope, sf = quant_rows(rows)
    pages = cache.size // page_stride
    for i, s in enumerate(slots):
        if 0 <= s < 64 * pages:
            page = cache[(s // 64) * page_stride + layer_off:][:MX8_PAGE]
            at = s % 64
            page[at * LATENT:(at + 1) * LATENT] = q[i]
            page[ROPE_AT + at * 128:ROPE_AT + (at + 1) * 128] = np.ascontiguousarray(rope[i]).view(np.uint8)
            page[SCALES_AT + at * 16:SCALES_AT + (at + 1) * 16] = sf[i]


def mx8_rows(cache, layer_off, page_stride, table, n):
    """Rows [n, 576] f64 of a block table; rows of pages that the cache does not hold are None in `held`."""
    pages = cache.size // page_stride
    out, held = np.zeros((n, ROW)), np.zeros(n, dtype=bool)
    for t in range(n):
        pid = int(table[t // 64])
        if not 0 <= pid < pages:
            continue
        page, at = cache[pid * page_stride + layer_off:][:MX8_PAGE], t % 64
        sc = page[SCALES_AT + at * 16:SCALES_AT + at * 16 + 16].astype(np.float64)
        sc = np.where(sc == 255, np.nan, 2.0 ** (sc - 127))
        out[t, :LATENT] = (_E4M3[page[at * LATENT:(at + 1) * LATENT]].reshape(16, 32) * sc[:, None]).reshape(-1)
        out[t, LATENT:] = k3o.bf16_to_f32(np.ascontiguousarray(page[ROPE_AT + at * 128:ROPE_AT + at * 128 + 128]).view(np.uint16))
        held[t] = True
    return out, held


def bf16_rows(cache, layer_off, page_stride, table, n):
    """The same of a flat bf16 cache (u16 bits; offsets in elements)."""
    pages = cache.size // page_stride
    out, held = np.zeros((n, ROW)), np.zeros(n, dtype=bool)
    for t in range(n):
        pid = int(table[t // 64])
        if 0 <= pid < pages:
            o = pid * page_stride + layer_off + (t % 64) * ROW
            out[t], held[t] = k3o.bf16_to_f32(cache[o:o + ROW]), True
    return out, held


def attn_oracle(q, rows_of, prefix_table, prefix_len, tables, lens, scale):
    """q [B, S, heads, 576] f64 -> (out, spread, ds): the output, sum_j p_j |v_j| per element, and the largest
    scale * sum |q| |k| of a row (what a rounding of its scores is relative to).  rows_of(table, n) -> (rows, held)."""
    B, S, H, _ = q.shape
    out, spread, ds = np.zeros((B, S, H, LATENT)), np.zeros((B, S, H, LATENT)), np.zeros((B, S, H))
    pn = min(prefix_len, 64 * len(prefix_table)) if prefix_table is not None else 0
    pk, ph = rows_of(prefix_table, max(0, pn)) if pn > 0 else (np.zeros((0, ROW)), np.zeros(0, dtype=bool))
    for b in range(B):
        if lens[b] < 0:
            continue
        n = min(int(lens[b]), 64 * tables.shape[1])
        sk, sh = rows_of(tables[b], n) if n else (np.zeros((0, ROW)), np.zeros(0, dtype=bool))
        for s in range(S):
            m = max(0, n - (S - 1 - s))
            k = np.concatenate([pk[ph], sk[:m][sh[:m]]])
            if not len(k):
                continue
            if not np.isfinite(k).all():
                out[b, s] = np.nan
                continue
            x = scale * (q[b, s] @ k.T)
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[b, s], spread[b, s] = p @ k[:, :LATENT], p @ np.abs(k[:, :LATENT])
            ds[b, s] = abs(scale) * (np.abs(q[b, s]) @ np.abs(k).T).max(1)
    return out, spread, ds


def attn_tolerance(out, spread, ds):
    """How far the kernel may be from the oracle, element by element.
      out: one rounding to bf16, half a step: 2^-8 |out|;
      the probabilities are rounded to bf16 for the matrix product: 2^-8 of each term, 2^-8 * sum p |v| in all;
      a score is a sum of 576 products in f32, each addition off by 2^-24 of a partial sum that sum |q| |k| bounds: 576 * 2^-24 * ds,
      with the scaling, the maximum's subtraction and the exponential's 2 ulp another 2^-22 of a score's size and 2^-21; an error d of the scores moves each
      p by a factor within exp(+-2 d), so the output by at most 2 d sum p |v| (3 d for d up to 0.1);
      sums over tokens in f32: tokens * 2^-24 of sum p |v|, below 2^-10 for 16384 tokens."""
    d = (ds * (576 * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -21)[..., None]
    assert np.all(d < 0.1)
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -8 + 2.0 ** -10 + 3 * d) * spread + 1e-30


def mx8_range_tolerance(q, rows_of, prefix_table, prefix_len, tables, lens, scale):
    """What k3g_latent_attn may lose beside attn_tolerance because MXFP8 pages and queries are multiplied as f16: (of the outputs, of the
    scores), per row.  M is the largest latent magnitude of the 16 tokens around one.
      an element below 2^-31 M may count as 0, one that does not is off by less: 2^-31 sum_j p_j M_j in the outputs, scale * 2^-31 M
      sum |q| in a score;
      a token's weight is off by 2^-25 where the largest weight * 2^E is 2^10 or more, and M is in (224, 448] 2^E: 2^-34 max_j p_j M_j for
      each token (twice that where E is what a neighbour's block, rounded up to it, gives);
      a query's element below 2^-39 of its row's largest may count as 0: scale * 2^-39 max |q| sum |k| in a score."""
    B, S, H, _ = q.shape
    lost, dlost = np.zeros((B, S, H)), np.zeros((B, S, H))

    def read(table, n):
        k, held = rows_of(table, n)
        big = np.zeros(n)
        for t in range(0, n, 16):
            big[t:t + 16] = np.abs(k[t:t + 16, :LATENT]).max()
        return k[held], big[held]
    empty = np.zeros((0, ROW)), np.zeros(0)
    pk, pm = read(prefix_table, prefix_len) if prefix_len > 0 else empty
    for b in range(B):
        sk, sm = read(tables[b], int(lens[b])) if lens[b] > 0 else empty
        for s in range(S):
            n = max(0, int(lens[b]) - (S - 1 - s))
            k, m = np.concatenate([pk, sk[:n]]), np.concatenate([pm, sm[:n]])
            if not len(k):
                continue
            x = scale * (q[b, s] @ k.T)
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            lost[b, s] = 2.0 ** -31 * (p @ m) + 2.0 ** -33 * len(k) * (p * m).max(1)
            lat = np.abs(q[b, s, :, :LATENT])
            dlost[b, s] = abs(scale) * (2.0 ** -31 * m.max() * lat.sum(1) + 2.0 ** -39 * lat.max(1) * np.abs(k[:, :LATENT]).sum(1).max())
    return lost, dlost


def verify_oracle(target, draft, ids, u):
    """(accepted, tokens) of k3g_verify_draft; target [B, S + 1, V], draft [B, S, V] or None."""
    B, S = ids.shape
    V = target.shape[2]
    accepted, tokens = np.zeros(B, dtype=np.int32), np.full((B, S + 1), -1, dtype=np.int64)

    def weights(x):
        with np.errstate(invalid="ignore"):
            return np.where((x > 0) & np.isfinite(x), x, 0.0)
    for b in range(B):
        kept, down = 0, False
        while kept < S and 0 <= ids[b, kept] < V:
            x = ids[b, kept]
            qx = float(draft[b, kept, x]) if draft is not None else 1.0
            if not float(u[b, kept]) * qx < float(target[b, kept, x]):
                down = True
                break
            kept += 1
        p = target[b, kept].astype(np.float64)
        w = weights(p)
        if down:
            q = draft[b, kept].astype(np.float64) if draft is not None else (np.arange(V) == ids[b, kept]).astype(np.float64)
            with np.errstate(invalid="ignore"):
                r = weights(p - q)
            w = r if r.sum() > 0 else w
        c = np.cumsum(w)
        pick = -1
        if c[-1] > 0:
            over = np.nonzero((c > float(u[b, S]) * c[-1]) & (w > 0))[0]
            pick = over[0] if len(over) else np.nonzero(w > 0)[0][-1]
        accepted[b] = kept
        tokens[b, :kept] = ids[b, :kept]
        tokens[b, kept] = pick
    return accepted, tokens
