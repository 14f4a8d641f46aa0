"""Cases and plain forms of the paged, tree-drafted decoding operators.

Four operators make up one step of decoding with drafted token trees over a
paged INT8 cache: the plan (block tables, slot maps, positions and ancestor
masks from request lengths), the write of new K/V rows into their pages, the
integer attention of the drafted tokens over the cache, and the log
probabilities of given tokens with entropy and top alternatives.

``run`` computes them in elementary torch operations where ``own`` is false,
and calls ``i_whisper_b200.ops`` where it is true.
"""
import math
import random

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a few live requests: the call's latency is all there is
        dict(name="plan_step_b8", op="plan", B=8, ctx_lo=0, ctx_hi=440, new_lo=1, new_hi=7, page=16, tree=True),
        # a full server: a thousand requests, each with a drafted tree
        dict(name="plan_trees_b1024", op="plan", B=1024, ctx_lo=1, ctx_hi=2000, new_lo=16, new_hi=64, page=32, tree=True),
        # one token of 256 utterances, K and V taken from the fused QKV rows of a 1024-wide decoder
        dict(name="write_step_b256", op="write", N=256, Hkv=16, D=64, page=16, pages=1024, pad=True),
        # prompts of many requests at once, 20 heads, an odd token count
        dict(name="write_prompts", op="write", N=40001, Hkv=20, D=64, page=32, pages=1400, pad=False),
        # the first drafted tokens of one utterance on a 6-head decoder: latency
        dict(name="tree_first_b1", op="attn", B=1, Hkv=6, G=1, D=64, page=16, ctx_lo=5, ctx_hi=5, new_lo=7, new_hi=7,
             tree=True, mult=70, shift=6, fb=13),
        # single-token decoding of 256 utterances anywhere in a 448-token text context
        dict(name="decode_b256", op="attn", B=256, Hkv=16, G=1, D=64, page=16, ctx_lo=0, ctx_hi=447, new_lo=1, new_hi=1,
             tree=False, mult=70, shift=6, fb=13),
        # drafted trees of 5 to 32 tokens for 64 utterances
        dict(name="trees_b64", op="attn", B=64, Hkv=16, G=1, D=64, page=16, ctx_lo=64, ctx_hi=416, new_lo=5, new_hi=32,
             tree=True, mult=70, shift=6, fb=14),
        # a decoder with shared key heads, wide heads and long contexts, trees of up to 64 tokens: the most arithmetic
        dict(name="trees_shared_heads", op="attn", B=16, Hkv=8, G=4, D=128, page=32, ctx_lo=1000, ctx_hi=8191, new_lo=24,
             new_hi=64, tree=True, mult=70, shift=7, fb=13),
        # single tokens over contexts that do not fit one block's shared memory: the most bytes
        dict(name="decode_long", op="attn", B=7, Hkv=20, G=1, D=64, page=16, ctx_lo=4097, ctx_hi=32700, new_lo=1, new_hi=1,
             tree=False, mult=100, shift=7, fb=13),
        # int8 classifier rows of a handful of utterances, best five alternatives: latency
        dict(name="logprobs_int8_b5", op="logp", N=5, V=51865, ld=51872, kind="int8", C=1, K=5, suppress=True),
        # rescoring of whole transcripts: every position of many hypotheses, int8 logits
        dict(name="logprobs_int8_rescore", op="logp", N=4096, V=51865, ld=51872, kind="int8", C=1, K=5, suppress=False),
        # sixteen-bit logits of a larger, odd vocabulary, several given tokens and twenty alternatives a row
        dict(name="logprobs_bf16", op="logp", N=1031, V=100003, ld=100003, kind="bfloat16", C=3, K=20, suppress=True),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "attn", "attn", "attn", "logp", "logp"])
    if op == "plan":
        B = _log(rng, 1, 2048)
        tree = rng.random() < 0.6
        hi = _log(rng, 1, 64) if tree else _log(rng, 1, max(2, 60000 // B))
        return dict(op=op, B=B, ctx_lo=0, ctx_hi=_log(rng, 1, 4000), new_lo=rng.randint(0, 1), new_hi=hi,
                    page=rng.choice([8, 16, 32, 64]), tree=tree)
    if op == "write":
        Hkv = rng.choice([1, 2, 6, 8, 12, 16, 20])
        D = rng.choice([64, 64, 128])
        N = _log(rng, 1, 40000 * 20 * 64 // (Hkv * D) if Hkv * D > 20 * 64 else 40000)
        page = rng.choice([8, 16, 32, 64])
        return dict(op=op, N=N, Hkv=Hkv, D=D, page=page, pages=N // page + rng.randint(2, 40), pad=rng.random() < 0.5)
    if op == "attn":
        while True:
            B, Hkv, G = _log(rng, 1, 256), rng.choice([1, 2, 6, 8, 12, 16, 20]), rng.choice([1, 1, 1, 2, 4, 8])
            D, page = rng.choice([64, 64, 64, 128]), rng.choice([8, 16, 32, 64])
            hi, new = _log(rng, 1, 32700), rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 64)])
            scores = B * Hkv * G * new * hi
            if scores <= 120_000_000 and B * Hkv * D * hi <= 220_000_000:
                break
        long = hi > 2000 or D == 128
        return dict(op=op, B=B, Hkv=Hkv, G=G, D=D, page=page, ctx_lo=rng.choice([0, hi // 3, hi]), ctx_hi=hi,
                    new_lo=rng.choice([1, new, (new + 1) // 2]), new_hi=new, tree=new > 1 and rng.random() < 0.7,
                    mult=rng.randint(60, 110), shift=7 if long else 6, fb=rng.choice([12, 13, 13, 14, 14, 15]))
    kind = rng.choice(["int8", "int8", "float16", "bfloat16", "float32"])
    size = {"int8": 1, "float16": 2, "bfloat16": 2, "float32": 4}[kind]
    V = rng.choice([51865, 51866, _log(rng, 40, 260000), _log(rng, 1000, 260000)])
    N = _log(rng, 1, max(1, min(8192, 206_000_000 // (V * size))))
    ld = rng.choice([V, (V + 31) // 32 * 32])
    return dict(op=op, N=N, V=V, ld=ld, kind=kind, C=rng.choice([0, 1, 1, 4]), K=min(V, rng.choice([0, 1, 5, 20, 32])),
                suppress=rng.random() < 0.4)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case):
    """Context and new lengths of every request: fixed by the case's sizes, so that work() knows them."""
    r = random.Random(repr([case[k] for k in ("B", "ctx_lo", "ctx_hi", "new_lo", "new_hi", "page")]))
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["B"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    ctx[-1], new[-1] = case["ctx_hi"], case["new_hi"]  # the longest is among them
    return ctx, new


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _normal8(g, sd, *shape, mean=0.0):
    x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16) * sd + mean
    return x.round_().clamp_(-127, 127).to(torch.int8)


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _parents(g, new):
    """A random drafted tree for each request: token i hangs from an earlier token of the request or from its
    context (-1), the first from the context."""
    n = sum(new)
    t = torch.arange(n, device=DEV) - torch.repeat_interleave(_i32(_starts(new)[:-1]), _i32(new), output_size=n)
    u = torch.rand(n, generator=g, device=DEV)
    return ((u * (t + 1)).floor().clamp(max=t) - 1).to(torch.int32)


def _pages(case, ctx, new, extra):
    page = case["page"]
    return sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + extra


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "plan":
        ctx, new = _lens(case)
        page, N = case["page"], sum(new)
        total = _pages(case, ctx, new, 64)
        width = max(-(-(c + n) // page) for c, n in zip(ctx, new))
        perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.full((case["B"], width), -1, dtype=torch.int32, device=DEV)
        have = [-(-c // page) for c in ctx]
        held = sum(have)
        rows = torch.repeat_interleave(torch.arange(case["B"], device=DEV), _i32(have), output_size=held)
        cols = torch.arange(held, device=DEV) - torch.repeat_interleave(_i32(_starts(have)[:-1]), _i32(have), output_size=held)
        table[rows, cols] = perm[:held]
        s.update(ctx=_i32(ctx), new=_i32(new), table=table, free=perm, head=_i32([held]), n=N, max_tokens=N + N // 16 + 3)
        if case["tree"]:
            par = torch.full((s["max_tokens"],), -1, dtype=torch.int32, device=DEV)
            par[:N] = _parents(g, new)
            s.update(parents=par, max_new=case["new_hi"])
        return s
    if op == "write":
        N, H, D = case["N"], case["Hkv"], case["D"]
        qkv = _normal8(g, 30, N, 3 * H * D)  # rows of the fused projection: K and V are columns of it
        s["k"], s["v"] = qkv[:, H * D:2 * H * D].view(N, H, D), qkv[:, 2 * H * D:].view(N, H, D)
        s["kc"] = _normal8(g, 30, case["pages"], H, case["page"], D)
        s["vc"] = _normal8(g, 30, case["pages"], H, case["page"], D)
        slots = torch.randperm(case["pages"] * case["page"], generator=g, device=DEV)[:N]
        if case["pad"]:  # padding rows of a captured step
            slots[N - N // 8:] = -1
        s["slots"] = slots
        return s
    if op == "attn":
        ctx, new = _lens(case)
        page, Hkv, D, H = case["page"], case["Hkv"], case["D"], case["Hkv"] * case["G"]
        N = sum(new)
        total = _pages(case, ctx, new, 3)
        width = max(-(-(c + n) // page) for c, n in zip(ctx, new))
        perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        cnt = [-(-(c + n) // page) for c, n in zip(ctx, new)]
        held = sum(cnt)
        table = torch.full((case["B"], width), -1, dtype=torch.int32, device=DEV)
        rows = torch.repeat_interleave(torch.arange(case["B"], device=DEV), _i32(cnt), output_size=held)
        cols = torch.arange(held, device=DEV) - torch.repeat_interleave(_i32(_starts(cnt)[:-1]), _i32(cnt), output_size=held)
        table[rows, cols] = perm[:held]
        s.update(ctx=_i32(ctx), starts=_i32(_starts(new)), table=table, tmax=case["new_hi"])
        qkv = _normal8(g, 30, N, (H + 2 * Hkv) * D)
        s["q"] = qkv[:, :H * D].view(N, H, D)
        s["kc"] = _normal8(g, 30, total, Hkv, page, D)
        # values differ by head and channel, as a projection's do: means over many keys stay away from zero
        mean = torch.randn(Hkv, 1, D, generator=g, device=DEV, dtype=torch.float16) * 18
        s["vc"] = _normal8(g, 25, total, Hkv, page, D, mean=mean)
        s["mask"] = None
        if case["tree"]:
            s["mask"] = _tree_bits(_parents(g, new), _i32(new), s["starts"], case["new_hi"], N)[0]
        return s
    N, V, ld, kind = case["N"], case["V"], case["ld"], case["kind"]
    if kind == "int8":
        x = _normal8(g, 25, N, ld)
        s["scale"] = 0.125
    else:
        x = torch.empty(N, ld, dtype=getattr(torch, kind), device=DEV).normal_(0, 3, generator=g)
        s["scale"] = 1.0
    s["x"] = x[:, :V]
    t = torch.randint(0, V, (N, case["C"]), generator=g, device=DEV)
    if case["C"] > 1:
        t[:, -1] = torch.where(torch.rand(N, generator=g, device=DEV) < 0.3, -1, t[:, -1])  # padded lists
    s["targets"] = t
    s["suppress"] = None
    if case["suppress"]:
        b = torch.rand((V + 31) // 32, 32, generator=g, device=DEV) < 0.02
        s["suppress"] = _pack32(b)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _pack32(bits):
    """[..., 32] truth values -> [...] int32 words, bit j of a word from place j."""
    w = (bits.to(torch.int64) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _tree_bits(parents, new, starts, tmax, N):
    """Ancestor-or-self bits [N, W] and depths [N] of ragged trees given by parent indices."""
    B = new.numel()
    req = torch.repeat_interleave(torch.arange(B, device=DEV), new, output_size=N)
    t = torch.arange(N, device=DEV) - starts[req]
    W = (tmax + 31) // 32
    up = torch.zeros(B, tmax, tmax + 1, device=DEV)
    up[req, t, torch.where(parents < 0, tmax, parents).long()] = 1.0  # column tmax: the context
    step = up[:, :, :tmax] + torch.eye(tmax, device=DEV)
    anc = (torch.linalg.matrix_power(step, tmax) > 0)[req, t]
    depth = anc.sum(1) - 1
    anc = torch.nn.functional.pad(anc, (0, 32 * W - tmax))
    return _pack32(anc.view(N, W, 32)), depth


def _plain_plan(s):
    ctx, new, table, free, head, page, M = (s["ctx"], s["new"], s["table"], s["free"], s["head"], s["case"]["page"],
                                            s["max_tokens"])
    B, width = table.shape
    F = free.numel()
    have, want = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    need = (want.clamp(max=width) - have).clamp(min=0)
    off = need.cumsum(0, dtype=torch.int32) - need
    col = torch.arange(width, device=DEV)
    j = col - have[:, None]
    at = head + off[:, None] + j
    granted = torch.where(at < F, free[at.clamp(0, F - 1).long()], -1)
    table.copy_(torch.where((j >= 0) & (j < need[:, None]), granted, table))
    starts = torch.nn.functional.pad(new.cumsum(0, dtype=torch.int32), (1, 0))
    i = torch.arange(M, device=DEV, dtype=torch.int32)
    live = i < starts[-1]
    req = torch.searchsorted(starts[1:], i, right=True).clamp(max=B - 1)
    t = i - starts[req]
    pos = ctx[req] + t
    c = pos // page
    pg = torch.where(c < width, table[req, c.clamp(max=width - 1).long()], -1)
    slot = torch.where(live & (pg >= 0), pg.long() * page + pos % page, -1)
    total = head + need.sum(dtype=torch.int32)
    status = (total > F).int() + 2 * (want > width).any().int() + 4 * (starts[-1] > M).int()
    out = dict(slots=slot, request=torch.where(live, req, -1).to(torch.int32), starts=starts, table=table,
               free_head=total.clamp(max=F), status=status)
    if s["case"]["tree"]:
        N = s["n"]
        bits, depth = _tree_bits(s["parents"][:N], new, starts, s["max_new"], N)
        out["mask"] = torch.nn.functional.pad(bits, (0, 0, 0, M - N))
        pos = torch.nn.functional.pad((ctx[req[:N]] + depth).to(torch.int32), (0, M - N))
        out["position"] = pos
    else:
        out["position"] = torch.where(live, pos, 0).to(torch.int32)
    return out


def _plain_write(s):
    k, v, slots, kc, vc, page = s["k"], s["v"], s["slots"], s["kc"], s["vc"], s["case"]["page"]
    dead = slots < 0  # written again as the first row, which is live
    slot = torch.where(dead, slots[0], slots)
    pg, off = slot // page, slot % page
    kc[pg, :, off] = torch.where(dead[:, None, None], k[0], k)
    vc[pg, :, off] = torch.where(dead[:, None, None], v[0], v)
    return dict(k_cache=kc, v_cache=vc)


def _rrs(x, s):
    """Rounding shift right, halves away from zero, in wrapping 32 bits."""
    if s <= 0:
        return x
    if s >= 32:
        return torch.zeros_like(x)
    half = 1 << (s - 1)
    half = half - (1 << 32) if half >= 1 << 31 else half
    return (x + half + (x >> 31)) >> s


def _w16(x):
    return ((x + 32768) & 65535) - 32768


def _shift_exp(x, xm, fb):
    """The int16 shift exponential 2^(x - xm) of the integer softmax, as 8 bits."""
    xs = _w16(x - xm)
    fix = _w16(_w16(xs + (xs >> 1)) - (xs >> 4))
    xi = fix >> fb
    fr = _w16(fix - _w16(xi << fb))
    num = _w16((1 << fb) + (fr >> 1))
    es = (-xi).clamp(0, 31)
    e = torch.where((xi > 0) | (es >= 16), 0, num >> es.clamp(max=15))
    e = (e >> (fb - 7) if fb > 7 else e) & 255
    return torch.where(xs > 0, 0, e)


def _fisr(x, off):
    """Integer reciprocal square root in Q(off): exponent-halving seed, two Newton steps, wrapping 32 bits."""
    e = torch.frexp(x.clamp(min=1).double())[1].to(torch.int32) - 1
    sig = torch.where(e <= 23, x << (23 - e).clamp(min=0), x >> (e - 23).clamp(min=0))
    bits = torch.where(x == 0, 0, ((e + 127) << 23) | (sig & 0x7FFFFF))
    bits = 0x5F3759DF - (bits >> 1) + (off << 23)
    e = ((bits >> 23) & 255) - 127
    sig = (bits & 0x7FFFFF) | 0x800000
    y = torch.where(e < 0, 0, torch.where(e >= 23, sig << (e - 23).clamp(0, 31), sig >> (23 - e).clamp(0, 31)))
    y = torch.where(e - 23 >= 32, 0, y)

    def newton(y):
        t = _rrs(x * y, off) * y
        return _rrs(y * ((3 << off) - t), off + 1)

    return newton(newton(y))


def _plain_attn(s):
    c = s["case"]
    q, kc, vc, table, ctx, starts, mask, T = (s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"], s["mask"],
                                              s["tmax"])
    N, H, D = q.shape
    B, width = table.shape
    Hkv, page = kc.shape[1], kc.shape[2]
    G, L = H // Hkv, width * page
    L256 = (L + 255) // 256 * 256
    new = starts[1:] - starts[:-1]
    req = torch.repeat_interleave(torch.arange(B, device=DEV), new, output_size=N)
    t = torch.arange(N, device=DEV) - starts[req]

    def rows(cache):  # [B, Hkv, L256, D]
        x = cache[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, D).float()
        return torch.nn.functional.pad(x, (0, 0, 0, L256 - L))

    qp = torch.zeros(B, T, H, D, device=DEV)
    qp[req, t] = q.float()
    qp = qp.view(B, T, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * T, D)
    key = torch.arange(L256, device=DEV)
    rel = key - ctx[:, None]  # [B, L256]: place among the new tokens
    if mask is None:
        seen = rel[:, None] <= torch.arange(T, device=DEV)[:, None]
    else:
        wp = torch.zeros(B, T, mask.shape[1], dtype=torch.int32, device=DEV)
        wp[req, t] = mask
        at = rel.clamp(0, 32 * mask.shape[1] - 1)[:, None].expand(B, T, L256)
        bit = (torch.gather(wp, 2, at >> 5) >> (at & 31)) & 1
        seen = (rel[:, None] < 0) | (bit != 0)
    seen = seen & (rel < new[:, None])[:, None]
    seen = seen[:, None, None].expand(B, 1, G, T, L256).reshape(B, 1, G * T, L256)
    x = torch.matmul(qp, rows(kc).transpose(2, 3)).int()  # exact: every partial sum is a whole number below 2^24
    x = _rrs(x * c["mult"], c["shift"]).clamp(-32768, 32767)
    m = torch.where(seen, x, -32768).amax(-1, keepdim=True)
    p = torch.where(seen, _shift_exp(x, m + 1, c["fb"]), 0)
    total = p.sum(-1, dtype=torch.int32)
    p = p.float().view(B, Hkv, G * T, L256 // 256, 256).transpose(2, 3)
    acc = torch.matmul(p, rows(vc).view(B, Hkv, L256 // 256, 256, D)).int().sum(2, dtype=torch.int32)
    inv = _fisr(total, 16)[..., None]
    o = _rrs(_rrs(_rrs(acc * inv, 16) * inv, 16) * 88, 5).clamp(-127, 127).to(torch.int8)
    o = o.view(B, Hkv, G, T, D).permute(0, 3, 1, 2, 4)[req, t]
    return o.reshape(N, H * D)


def _plain_logp(s):
    x, tg, K, scale = s["x"].float(), s["targets"], s["case"]["K"], s["scale"]
    N, V = x.shape
    if s["suppress"] is not None:
        bits = (s["suppress"][:, None] >> torch.arange(32, device=DEV)) & 1
        x = torch.where(bits.view(-1)[:V] != 0, -math.inf, x)
    l = x * scale
    m = l.amax(1, keepdim=True)
    e = torch.exp(l - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    entropy = torch.log(total[:, 0]) - torch.where(e > 0, e * (l - m), 0).sum(1) / total[:, 0]
    lp = torch.gather(l, 1, tg.clamp(min=0)) - lse
    lp = torch.where(tg < 0, 0, lp)
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    val, idx = val[:, :K], idx[:, :K]
    gone = val == -math.inf
    top = torch.where(gone, -math.inf, val * scale - lse)
    return dict(logprobs=lp, entropy=entropy, top_ids=torch.where(gone, -1, idx), top_logprobs=top)


def _own(s):
    from i_whisper_b200 import ops
    c = s["case"]
    if c["op"] == "plan":
        p = ops.paged_plan_cuda(s["ctx"], s["new"], s["table"], s["free"], s["head"], c["page"], s["max_tokens"],
                                parents=s.get("parents"), max_new=s.get("max_new"))
        out = dict(slots=p.slots, request=p.request, starts=p.starts, table=s["table"], free_head=p.free_head,
                   status=p.status, position=p.position)
        if c["tree"]:
            out["mask"] = p.tree_mask
        return out
    if c["op"] == "write":
        ops.paged_kv_write_cuda(s["k"], s["v"], s["slots"], s["kc"], s["vc"])
        return dict(k_cache=s["kc"], v_cache=s["vc"])
    if c["op"] == "attn":
        return ops.tree_attention_cuda(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["starts"], c["mult"], c["shift"],
                                       c["fb"], 88, 5, rsqrt_offset=16, tree_mask=s["mask"])
    lp, entropy, ids, top = ops.token_logprobs_cuda(s["x"], s["targets"], top=c["K"], scale=s["scale"],
                                                    suppress_bits=s["suppress"])
    return dict(logprobs=lp, entropy=entropy, top_ids=ids, top_logprobs=top)


def run(s):
    if own:
        return _own(s)
    return {"plan": _plain_plan, "write": _plain_write, "attn": _plain_attn, "logp": _plain_logp}[s["case"]["op"]](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        ctx, new = _lens(case)
        N, page = sum(new), case["page"]
        M = N + N // 16 + 3
        fresh = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(ctx, new))
        words = (case["new_hi"] + 31) // 32 if case["tree"] else 0
        return {"bytes": 12 * case["B"] + 8 * fresh + M * (16 + 4 * words) + (4 * N if case["tree"] else 0), "flops": 0}
    if op == "write":
        live = case["N"] - (case["N"] // 8 if case["pad"] else 0)
        return {"bytes": 4 * live * case["Hkv"] * case["D"] + 8 * case["N"], "flops": 0}
    if op == "attn":
        ctx, new = _lens(case)
        Hkv, H, D = case["Hkv"], case["Hkv"] * case["G"], case["D"]
        keys = sum(c + n for c, n in zip(ctx, new) if n)
        pairs = sum(n * (c + n) for c, n in zip(ctx, new))
        return {"bytes": 2 * keys * Hkv * D + 2 * sum(new) * H * D, "flops": 4 * pairs * H * D}
    size = {"int8": 1, "float16": 2, "bfloat16": 2, "float32": 4}[case["kind"]]
    N, V = case["N"], case["V"]
    return {"bytes": N * V * size + N * (12 * case["C"] + 4 + 12 * case["K"]) + (V // 8 if case["suppress"] else 0),
            "flops": 4 * N * V}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, request by request and row by row
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "attn":
        return _exact_attn(prepare(case, seed))
    if case["op"] == "logp":
        return _exact_logp(prepare(case, seed))
    return None  # tables and copies: whole numbers, compared bit for bit with the plain form


def _exact_attn(s):
    c = s["case"]
    N, H, D = s["q"].shape
    page, Hkv = c["page"], c["Hkv"]
    G = H // Hkv
    starts, ctx = s["starts"].tolist(), s["ctx"].tolist()
    out = torch.zeros(N, H, D, dtype=torch.int8, device=DEV)
    lo, hi = -32768, 32767

    def i16(x):
        return (x - lo) % 65536 + lo

    def i32(x):
        return (x + 2 ** 31) % 2 ** 32 - 2 ** 31

    def shift(x, n):  # halves away from zero
        return torch.sign(x) * ((x.abs() + (1 << (n - 1))) >> n) if n > 0 else x

    for b in range(c["B"]):
        a, z, L = starts[b], starts[b + 1], ctx[b] + starts[b + 1] - starts[b]
        if a == z:
            continue
        pages = s["table"][b, :-(-L // page)].long()
        k = s["kc"][pages].transpose(1, 2).reshape(-1, Hkv, D)[:L].double()
        v = s["vc"][pages].transpose(1, 2).reshape(-1, Hkv, D)[:L].double()
        q = s["q"][a:z].double().view(z - a, Hkv, G, D)
        j = torch.arange(z - a, device=DEV)
        if s["mask"] is None:
            near = j[None] <= j[:, None]
        else:
            near = (s["mask"][a:z].long()[:, j // 32] >> (j % 32)) % 2 == 1
        open_ = torch.cat([torch.ones(z - a, ctx[b], dtype=torch.bool, device=DEV), near], 1)[None, None]
        x = torch.einsum("thgd,lhd->hgtl", q, k).long() * c["mult"]
        x = shift(x, c["shift"]).clamp(lo, hi)
        m = x.masked_fill(~open_, lo).amax(-1, keepdim=True)
        d = i16(x - i16(m + 1))
        f = i16(i16(d + torch.div(d, 2, rounding_mode="floor")) - torch.div(d, 16, rounding_mode="floor"))
        whole = torch.div(f, 1 << c["fb"], rounding_mode="floor")
        part = i16(f - i16(whole * (1 << c["fb"])))
        mant = i16((1 << c["fb"]) + torch.div(part, 2, rounding_mode="floor"))
        val = torch.div(mant, 2 ** (-whole).clamp(0, 40), rounding_mode="floor")
        val = val.masked_fill((whole > 0) | (whole <= -16), 0)
        val = (torch.div(val, 1 << (c["fb"] - 7), rounding_mode="floor") if c["fb"] > 7 else val) % 256
        p = val.masked_fill((d > 0) | ~open_, 0)
        n = p.sum(-1)
        acc = i32(torch.einsum("hgtl,lhd->hgtd", p.double(), v).long())
        # reciprocal square root: seed from the exponent and truncated mantissa, two Newton steps
        ex = torch.frexp(n.clamp(min=1).double())[1].long() - 1
        man = torch.where(ex <= 23, n * 2 ** (23 - ex).clamp(min=0), torch.div(n, 2 ** (ex - 23).clamp(min=0), rounding_mode="floor"))
        word = torch.where(n == 0, 0, (ex + 127) * 2 ** 23 + man % 2 ** 23)
        word = 0x5F3759DF - torch.div(word, 2, rounding_mode="floor") + 16 * 2 ** 23
        ex = torch.div(word, 2 ** 23, rounding_mode="floor") % 256 - 127
        man = word % 2 ** 23 + 2 ** 23
        y = torch.where(ex >= 23, man * 2 ** (ex - 23).clamp(0, 31), torch.div(man, 2 ** (23 - ex).clamp(0, 40), rounding_mode="floor"))
        y = i32(torch.where(ex < 0, 0, y))
        for _ in range(2):
            r = i32(shift(i32(n * y), 16) * y)
            y = shift(i32(y * i32(3 * 2 ** 16 - r)), 17)
        y = y[..., None]
        o = shift(i32(shift(i32(shift(i32(acc * y), 16) * y), 16) * 88), 5).clamp(-127, 127)
        out[a:z] = o.permute(2, 0, 1, 3).reshape(z - a, H, D).to(torch.int8)
    return out.view(N, H * D)


def _exact_logp(s):
    K, N = s["case"]["K"], s["x"].shape[0]
    C = s["case"]["C"]
    lp = torch.zeros(N, C, dtype=torch.float64, device=DEV)
    ent = torch.zeros(N, dtype=torch.float64, device=DEV)
    top = torch.zeros(N, K, dtype=torch.float64, device=DEV)
    off = None
    if s["suppress"] is not None:
        v = torch.arange(s["x"].shape[1], device=DEV)
        off = (s["suppress"].long()[v // 32] >> (v % 32)) % 2 == 1
    for a in range(0, N, 256):
        z = s["x"][a:a + 256].double() * s["scale"]
        if off is not None:
            z = z.masked_fill(off, -math.inf)
        z = torch.log_softmax(z, 1)
        ent[a:a + 256] = -(z.exp() * z.masked_fill(z == -math.inf, 0)).sum(1)
        t = s["targets"][a:a + 256]
        lp[a:a + 256] = z.gather(1, t.clamp(min=0)).masked_fill(t < 0, 0)
        if K:
            top[a:a + 256] = z.topk(K, 1).values
    return dict(logprobs=lp, entropy=ent, top_ids=None, top_logprobs=top)
