"""Plain 64-bit implementations of the paged, tree-drafted decoding operators
(test helper): numpy, request by request and row by row, written from the
definitions in include/iwhisper_b200.h."""
import numpy as np


def _i16(x):
    return (x + 32768) % 65536 - 32768


def _i32(x):
    return (x + 2 ** 31) % 2 ** 32 - 2 ** 31


def rounding_rshift(x, s):
    """Halves away from zero; 0 -> x, 32 and more -> 0 (wrapping 32 bits)."""
    if s <= 0:
        return x
    if s >= 32:
        return np.zeros_like(x)
    return _i32(x + (1 << (s - 1)) - (x < 0)) >> s


def shift_exp(x, xm, fb):
    xs = _i16(x - xm)
    fix = _i16(_i16(xs + (xs >> 1)) - (xs >> 4))
    xi = fix >> fb
    fr = _i16(fix - _i16(xi << fb))
    num = _i16((1 << fb) + (fr >> 1))
    es = np.clip(-xi, 0, 63)
    e = np.where((xi > 0) | (es >= 16), 0, num >> np.minimum(es, 15))
    e = (e >> (fb - 7)) % 256 if fb > 7 else e % 256
    return np.where(xs > 0, 0, e)


def fisr(x, off):
    if x == 0:
        bits = 0
    else:
        e = int(x).bit_length() - 1
        sig = (x << (23 - e)) if e <= 23 else (x >> (e - 23))
        bits = ((e + 127) << 23) | (sig & 0x7FFFFF)
    bits = (0x5F3759DF - (bits >> 1) + (off << 23)) % 2 ** 32
    e = ((bits >> 23) & 255) - 127
    sig = (bits & 0x7FFFFF) | 0x800000
    y = 0 if e < 0 else _i32((sig << (e - 23)) if e >= 23 else (sig >> (23 - e)))
    for _ in range(2):
        a = np.int64(_i32(x * y))
        t = _i32(int(rounding_rshift(a, off)) * y)
        y = int(rounding_rshift(np.int64(_i32(y * _i32((3 << off) - t))), off + 1))
    return y


def tree_attention(q, k_cache, v_cache, table, ctx, starts, mult, shift, fb, av_mult, av_shift, off=16, mask=None):
    """[N, H, D] int8 queries -> [N, H*D] int8; caches [P, Hkv, page, D]."""
    N, H, D = q.shape
    P, Hkv, page, _ = k_cache.shape
    y = np.zeros((N, H, D), np.int8)
    for b in range(len(ctx)):
        c, a, z = max(int(ctx[b]), 0), int(starts[b]), int(starts[b + 1])
        L = min(c + z - a, table.shape[1] * page)
        there = np.array([0 <= table[b, j // page] < P for j in range(L)], bool)
        pg = np.array([table[b, j // page] if there[j] else 0 for j in range(L)], np.int64)
        row = np.arange(L) % page
        for n in range(a, z):
            u = np.arange(L) - c
            if mask is None:
                seen = u <= n - a
            else:
                w = mask.shape[1]
                bit = (mask[n, np.clip(u >> 5, 0, w - 1)].astype(np.int64) >> (u & 31)) & 1
                seen = (u < 0) | ((u >> 5 < w) & (bit == 1))
            seen &= there
            if not seen.any():
                continue
            for h in range(H):
                g = h // (H // Hkv)
                K, V = k_cache[pg, g, row].astype(np.int64), v_cache[pg, g, row].astype(np.int64)
                x = _i32((K @ q[n, h].astype(np.int64)) * mult)
                x = np.clip(rounding_rshift(x, shift), -32768, 32767)
                p = np.where(seen, shift_exp(x, _i16(x[seen].max() + 1), fb), 0)
                i = fisr(int(p.sum()), off)
                o = rounding_rshift(_i32(_i32(p @ V) * i), off)
                o = rounding_rshift(_i32(o * i), off)
                o = rounding_rshift(_i32(o * av_mult), av_shift)
                y[n, h] = np.clip(o, -127, 127)
    return y.reshape(N, H * D)


def paged_plan(ctx, new, table, free, head, page, max_tokens, parents=None, max_new=0, max_len=1 << 30):
    """-> dict of the plan's outputs with the new block table."""
    B, width = table.shape
    table = table.copy()
    status = 0
    words = (max_new + 31) // 32 if parents is not None else 0
    out = dict(slots=np.full(max_tokens, -1, np.int64), request=np.full(max_tokens, -1, np.int32),
               position=np.zeros(max_tokens, np.int32), starts=np.zeros(B + 1, np.int32),
               tree_mask=np.zeros((max_tokens, words), np.int64))
    head = min(max(int(head), 0), len(free))
    i = 0
    for b in range(B):
        c, n = int(ctx[b]), int(new[b])
        if not 0 <= c <= max_len:
            c, status = 0, status | 8
        if not 0 <= n <= max_len:
            n, status = 0, status | 8
        if words and n > max_new:
            status |= 16
        have, want = -(-c // page), -(-(c + n) // page)
        if want > width:
            status |= 2
        for col in range(have, min(want, width)):
            if head < len(free):
                table[b, col] = free[head]
                head += 1
            else:
                table[b, col] = -1
                status |= 1
        out["starts"][b] = min(i, 2 ** 31 - 1)
        first = i
        for t in range(min(n, max(0, max_tokens - first))):
            p = c + t
            pg = table[b, p // page] if p // page < width else -1
            out["slots"][i + t] = -1 if pg < 0 else int(pg) * page + p % page
            out["request"][i + t] = b
            depth, u = 0, t
            while words:
                if u >> 5 < words:
                    out["tree_mask"][i + t, u >> 5] |= 1 << (u & 31)
                up = int(parents[first + u])
                if not 0 <= up < u:
                    break
                u, depth = up, depth + 1
            out["position"][i + t] = c + (depth if words else t)
        i += n
    out["starts"][B] = min(i, 2 ** 31 - 1)
    if i > max_tokens:
        status |= 4
    out["tree_mask"] = _i32(out["tree_mask"]).astype(np.int32)
    return dict(out, table=table, free_head=head, status=status)


def token_logprobs(x, targets, top, scale, suppress=None):
    """float64 rows -> (logprobs, entropy, ids, top_logprobs); `suppress`: truth values [V]."""
    x = np.asarray(x, np.float64)
    N, V = x.shape
    C = targets.shape[1]
    lp, ent = np.zeros((N, C)), np.zeros(N)
    ids, tl = np.full((N, top), -1, np.int64), np.full((N, top), -np.inf)
    live = np.ones(V, bool) if suppress is None else ~suppress
    for n in range(N):
        l = np.where(live, x[n], -np.inf)
        bad = bool(np.isnan(l).any() or (l == np.inf).any())
        some = np.flatnonzero(l > -np.inf)
        if not bad and len(some):
            m = (l[some] * scale).max()
            e = np.exp(l[some] * scale - m)
            lse = m + np.log(e.sum())
            ent[n] = lse - (e * l[some] * scale).sum() / e.sum()
            order = some[np.lexsort((some, -l[some]))][:top]
            ids[n, :len(order)], tl[n, :len(order)] = order, l[order] * scale - lse
        elif bad:
            ent[n], tl[n] = np.nan, np.nan
        for c in range(C):
            t = targets[n, c]
            if t < 0:
                lp[n, c] = 0
            elif t >= V or bad:
                lp[n, c] = np.nan
            elif l[t] == -np.inf:
                lp[n, c] = -np.inf
            else:
                lp[n, c] = l[t] * scale - lse
    return lp, ent, ids, tl
