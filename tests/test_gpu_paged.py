"""The paged, tree-drafted decoding operators on the GPU against plain 64-bit
implementations (tests/paged_reference.py). Integer outputs are compared bit
for bit; the tolerance of the log probabilities is derived in `_lp_tol`."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from i_whisper_b200 import ops as _ops
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
def _check_plan(ops, ctx, new, page, width, n_free, head, max_tokens, parents=None, max_new=None, pad_cols=0):
    rng = np.random.default_rng(len(ctx) * 131 + page)
    B = len(ctx)
    table = rng.integers(0, 5000, (B, width + pad_cols)).astype(np.int32)
    free = rng.permutation(5000 + n_free)[:n_free].astype(np.int32)
    want = R.paged_plan(ctx, new, table[:, :width], free, head, page, max_tokens, parents, max_new or 0)
    t = dev(table)
    for _ in range(2):  # the same call again gives the same plan
        p = ops.paged_plan_cuda(dev(np.asarray(ctx, np.int32)), dev(np.asarray(new, np.int32)), t[:, :width], dev(free),
                                dev(np.asarray([head], np.int32)), page, max_tokens,
                                None if parents is None else dev(parents), max_new)
        for name in ("slots", "request", "position", "starts"):
            assert np.array_equal(getattr(p, name).cpu().numpy(), want[name]), name
        assert p.status.item() == want["status"] and p.free_head.item() == want["free_head"]
        assert np.array_equal(t[:, :width].cpu().numpy(), want["table"])
        assert np.array_equal(t[:, width:].cpu().numpy(), table[:, width:])
        if parents is not None:
            assert np.array_equal(p.tree_mask.cpu().numpy(), want["tree_mask"])
    return want["status"]


def _random_parents(rng, new, max_tokens, wild=False):
    par = np.full(max_tokens, -1, np.int32)
    i = 0
    for n in new:
        for t in range(n):
            if i + t < max_tokens:
                par[i + t] = rng.integers(-3, n + 2) if wild else rng.integers(-1, t) if t else -1
        i += max(n, 0)
    return par


@pytest.mark.parametrize("B,page,tree", [(1, 16, False), (1, 1, True), (3, 8, True), (33, 16, False), (257, 32, True),
                                         (700, 64, False), (1300, 16, True)])
def test_plan(ops, B, page, tree):
    rng = np.random.default_rng(B + page)
    ctx = rng.integers(0, 300, B).tolist()
    new = rng.integers(0, 41, B).tolist()
    if B > 2:
        ctx[1], new[1], new[2] = 0, 0, 1
    width = -(-400 // page)
    N = sum(new)
    par = _random_parents(rng, new, N + 5) if tree else None
    assert _check_plan(ops, ctx, new, page, width, 60 * B * 8 // page + 64 * B, 3, N + 5, par, 40 if tree else None) == 0


def test_plan_most_requests(ops):
    from i_whisper_b200 import _lib
    rng = np.random.default_rng(1)
    B = _lib.PLAN_MAX_REQUESTS
    ctx, new = rng.integers(0, 40, B).tolist(), rng.integers(0, 3, B).tolist()
    assert _check_plan(ops, ctx, new, 8, 6, 2 * B, 0, sum(new) + 1) == 0


def test_plan_first_call_around_the_default_shared_memory():
    """Request counts whose two sums alone fit the default 48 KB of shared memory, but not beside the kernel's own
    variables, as the first call of a process (later calls would find the limit raised)."""
    code = """
import torch
from i_whisper_b200 import ops
for B in (6125, 6126, 6143, 6144):
    one = torch.ones(B, dtype=torch.int32, device="cuda")
    p = ops.paged_plan_cuda(one, one, torch.zeros(B, 1, dtype=torch.int32, device="cuda"), one[:1], one[:1] * 0, 16, B)
    assert p.starts.tolist() == list(range(B + 1)) and p.slots.tolist() == [1] * B and p.status.item() == 0
print("ok")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def test_plan_chain_of_drafts_crosses_mask_words(ops):
    new = [70, 1, 64, 33]
    par = np.concatenate([np.arange(n, dtype=np.int32) - 1 for n in new])
    assert _check_plan(ops, [5, 0, 31, 32], new, 16, 9, 64, 0, sum(new), par, 70) == 0


def test_plan_reports_what_does_not_fit(ops):
    # free pages run out inside the second request; a table too short; too many tokens; bad lengths
    assert _check_plan(ops, [3, 16, 0], [20, 40, 5], 16, 6, 2, 0, 65) == 1
    assert _check_plan(ops, [3, 90, 0], [4, 20, 5], 16, 6, 9, 0, 29) == 2
    assert _check_plan(ops, [300, 90], [4, 3], 16, 6, 9, 0, 29) == 2
    assert _check_plan(ops, [3, 9, 0], [4, 20, 5], 16, 6, 9, 0, 7) == 4
    assert _check_plan(ops, [-5, 9, 2 ** 30 + 1], [4, -1, 5], 16, 6, 9, 0, 12) == 8
    assert _check_plan(ops, [3], [20], 16, 6, 9, 9, 20) == 1
    assert _check_plan(ops, [3], [20], 16, 6, 9, -4, 20) == 0
    assert _check_plan(ops, [3], [20], 16, 6, 9, 700, 20) == 1


def test_plan_bad_parents_and_large_trees(ops):
    rng = np.random.default_rng(0)
    new = [9, 40, 3]
    par = _random_parents(rng, new, 52, wild=True)
    assert _check_plan(ops, [1, 2, 3], new, 16, 6, 9, 0, 52, par, 32) == 16


def test_plan_sums_above_32_bits(ops):
    big = [2 ** 30] * 5
    B = len(big)
    free = torch.arange(7, dtype=torch.int32, device="cuda")
    t = torch.full((B, 4), -7, dtype=torch.int32, device="cuda")
    p = ops.paged_plan_cuda(dev(np.zeros(B, np.int32)), dev(np.asarray(big, np.int32)), t, free,
                            dev(np.zeros(1, np.int32)), 16, 40)
    assert p.starts.tolist() == [0, 2 ** 30] + [2 ** 31 - 1] * 4
    assert p.slots.tolist() == list(range(40))
    assert p.status.item() == 1 | 2 | 4
    assert t.cpu().tolist() == [[0, 1, 2, 3], [4, 5, 6, -1]] + [[-1] * 4] * 3


def test_plan_no_tokens_and_empty_pool(ops):
    assert _check_plan(ops, [0, 16, 7], [0, 0, 0], 16, 3, 1, 0, 0) == 0
    assert _check_plan(ops, [0, 16, 7], [1, 0, 1], 16, 3, 0, 0, 4) == 1


def test_plan_refusals(ops):
    i = lambda *v: dev(np.asarray(v, np.int32))
    t = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="power of two"):
        ops.paged_plan_cuda(i(1, 2), i(1, 1), t, i(1), i(0), 24, 2)
    with pytest.raises(RuntimeError, match="new_lens"):
        ops.paged_plan_cuda(i(1, 2), i(1), t, i(1), i(0), 16, 2)
    with pytest.raises(RuntimeError, match="block_table"):
        ops.paged_plan_cuda(i(1, 2), i(1, 1), t[:, ::2], i(1), i(0), 16, 2)
    with pytest.raises(RuntimeError, match="max_new"):
        ops.paged_plan_cuda(i(1, 2), i(1, 1), t, i(1), i(0), 16, 2, parents=i(-1, -1))
    with pytest.raises(RuntimeError, match="parents"):
        ops.paged_plan_cuda(i(1, 2), i(1, 1), t, i(1), i(0), 16, 2, parents=i(-1), max_new=1)
    with pytest.raises(RuntimeError, match="context_lens"):
        ops.paged_plan_cuda(i(1, 2).long(), i(1, 1), t, i(1), i(0), 16, 2)
    with pytest.raises(RuntimeError, match="current CUDA device"):
        ops.paged_plan_cuda(i(1, 2).cpu(), i(1, 1), t, i(1), i(0), 16, 2)


# ---------------------------------------------------------------------------
# cache write
# ---------------------------------------------------------------------------
def _cache(rng, P, H, page, D, order="phrd"):
    """Random cache [P, H, page, D] whose storage order of the axes is `order`."""
    sizes = dict(p=P, h=H, r=page, d=D)
    a = dev(rng.integers(-128, 128, [sizes[c] for c in order], dtype=np.int8))
    return a.permute([order.index(c) for c in "phrd"])


@pytest.mark.parametrize("N,H,D,page,order", [(1, 6, 64, 16, "phrd"), (37, 16, 64, 16, "prhd"), (129, 5, 128, 8, "hprd"),
                                              (4, 3, 16, 1, "phrd"), (1000, 20, 64, 64, "prhd")])
def test_kv_write(ops, N, H, D, page, order):
    rng = np.random.default_rng(N + H)
    P = -(-N // page) + 3
    qkv = dev(rng.integers(-128, 128, (N, 3 * H * D), dtype=np.int8))
    k, v = qkv[:, H * D:2 * H * D].view(N, H, D), qkv[:, 2 * H * D:].view(N, H, D)
    kc, vc = _cache(rng, P, H, page, D, order), _cache(rng, P, H, page, D, order)
    slots = rng.permutation(P * page)[:N].astype(np.int64)
    slots[::5] = -1
    if N > 3:
        slots[3] = P * page  # past the cache: skipped
    wk, wv = kc.cpu().numpy().copy(), vc.cpu().numpy().copy()
    for n in range(N):
        if 0 <= slots[n] < P * page:
            wk[slots[n] // page, :, slots[n] % page] = k[n].cpu().numpy()
            wv[slots[n] // page, :, slots[n] % page] = v[n].cpu().numpy()
    ops.paged_kv_write_cuda(k, v, dev(slots), kc, vc)
    assert np.array_equal(kc.cpu().numpy(), wk) and np.array_equal(vc.cpu().numpy(), wv)


def test_kv_write_head_order_and_empty(ops):
    rng = np.random.default_rng(9)
    k = dev(rng.integers(-128, 128, (4, 7, 64), dtype=np.int8)).transpose(0, 1)  # [7, 4, 64], head-major rows
    kc, vc = _cache(rng, 3, 4, 4, 64), _cache(rng, 3, 4, 4, 64)
    slots = dev(np.arange(7, dtype=np.int64) + 2)
    ops.paged_kv_write_cuda(k, k, slots, kc, vc)
    flat = kc.permute(0, 2, 1, 3).reshape(12, 4, 64)
    assert torch.equal(flat[2:9], k)
    before = kc.clone()
    ops.paged_kv_write_cuda(k[:0], k[:0], slots[:0], kc, vc)
    assert torch.equal(before, kc)


def test_kv_write_past_2_to_31_bytes(ops):
    """Slots whose byte offset does not fit 32 bits."""
    P, H, page, D = 2200, 16, 1024, 64  # 2.3 GB
    kc = torch.zeros(P, H, page, D, dtype=torch.int8, device="cuda")
    k = dev(np.random.default_rng(1).integers(-128, 128, (3, H, D), dtype=np.int8))
    slots = [5, 2 ** 31 // (H * D) + 77, P * page - 1]
    ops.paged_kv_write_cuda(k, k, dev(np.asarray(slots, np.int64)), kc, kc)
    for n, s in enumerate(slots):
        assert torch.equal(kc[s // page, :, s % page], k[n])
    assert kc.count_nonzero() == k.count_nonzero()


def test_kv_write_refusals(ops):
    k = torch.zeros(4, 2, 64, dtype=torch.int8, device="cuda")
    kc = torch.zeros(3, 2, 16, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="heads"):
        ops.paged_kv_write_cuda(k, k, s, kc[:, :1], kc[:, :1])
    with pytest.raises(RuntimeError, match="slots"):
        ops.paged_kv_write_cuda(k, k, s.int(), kc, kc)
    with pytest.raises(RuntimeError, match="power of two"):
        ops.paged_kv_write_cuda(k, k, s, kc[:, :, :12], kc[:, :, :12])
    with pytest.raises(RuntimeError, match="16-byte"):
        w = torch.zeros(4, 2, 72, dtype=torch.int8, device="cuda")[:, :, 8:]
        ops.paged_kv_write_cuda(w, w, s, kc, kc)
    with pytest.raises(RuntimeError, match="int8"):
        ops.paged_kv_write_cuda(k.short(), k.short(), s, kc, kc)
    with pytest.raises(RuntimeError, match="equal strides"):
        ops.paged_kv_write_cuda(k, k, s, kc, kc.transpose(1, 2).contiguous().transpose(1, 2))


# ---------------------------------------------------------------------------
# tree attention
# ---------------------------------------------------------------------------
def _attn_case(seed, ctx, new, Hkv, G, D, page, tree=True, sd=30, order="phrd", extra_width=0, empty_rows=False):
    rng = np.random.default_rng(seed)
    B, N, H = len(ctx), sum(new), Hkv * G
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    cnt = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    P = sum(cnt) + 3
    perm = rng.permutation(P).astype(np.int32)
    table = np.full((B, max(cnt + [1]) + extra_width), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, :cnt[b]] = perm[at:at + cnt[b]]
        at += cnt[b]
    gauss = lambda *s: np.clip(np.round(rng.normal(0, sd, s)), -128, 127).astype(np.int8)
    q, mask = gauss(N, H, D), None
    if tree:
        mask = np.zeros((N, (max(new) + 31) // 32 + 1), np.int64)
        for b in range(B):
            anc = []
            for t in range(new[b]):
                up = rng.integers(-1, t) if t else -1
                a = (anc[up] if up >= 0 else 0) | (1 << t)
                anc.append(a)
                if empty_rows and t % 3 == 1:
                    a = 0
                for w in range(mask.shape[1]):
                    mask[starts[b] + t, w] = (a >> (32 * w)) & 0xFFFFFFFF
        mask = ((mask + 2 ** 31) % 2 ** 32 - 2 ** 31).astype(np.int32)
    sizes = dict(p=P, h=Hkv, r=page, d=D)
    kc, vc = (gauss(*[sizes[c] for c in order]) for _ in range(2))
    axes = [order.index(c) for c in "phrd"]
    return dict(q=q, kc=kc, vc=vc, axes=axes, table=table, ctx=np.asarray(ctx, np.int32), starts=starts, mask=mask)


def _check_attn(ops, c, mult=70, shift=6, fb=13, av=(88, 5), off=16, out=None):
    kc, vc = dev(c["kc"]).permute(c["axes"]), dev(c["vc"]).permute(c["axes"])
    want = R.tree_attention(c["q"], c["kc"].transpose(c["axes"]), c["vc"].transpose(c["axes"]), c["table"], c["ctx"],
                            c["starts"], mult, shift, fb, *av, off, c["mask"])
    got = ops.tree_attention_cuda(dev(c["q"]), kc, vc, dev(c["table"]), dev(c["ctx"]), dev(c["starts"]), mult, shift, fb,
                                  *av, rsqrt_offset=off, tree_mask=None if c["mask"] is None else dev(c["mask"]), out=out)
    assert np.array_equal(got.cpu().numpy(), want)
    return got


@pytest.mark.parametrize("ctx,new,Hkv,G,D,page,tree", [
    ([0], [1], 1, 1, 64, 16, False),
    ([1], [1], 6, 1, 64, 1, True),
    ([5], [7], 6, 1, 64, 16, True),
    ([447, 0, 31, 32, 33], [1, 1, 1, 1, 1], 3, 1, 64, 16, False),
    ([100, 7, 250], [16, 17, 15], 2, 1, 64, 8, True),
    ([100, 0, 63, 1], [33, 64, 1, 0], 2, 1, 64, 32, True),
    ([40, 200], [5, 12], 2, 4, 128, 64, True),
    ([3, 129, 700], [1, 1, 1], 1, 8, 128, 16, False),
    ([513, 90], [20, 3], 1, 5, 64, 16, False),
    ([0, 0, 12], [65, 0, 40], 1, 1, 64, 4, True),
    ([1500], [3], 2, 1, 64, 128, False),
    ([2000, 1999, 2049], [9, 2, 1], 1, 2, 64, 16, True),
    ([1024, 990], [6, 31], 1, 2, 128, 16, True),
])
def test_tree_attention(ops, ctx, new, Hkv, G, D, page, tree):
    _check_attn(ops, _attn_case(len(ctx) * 7 + page, ctx, new, Hkv, G, D, page, tree))


@pytest.mark.parametrize("mult,shift,fb,av,off", [
    (118, 8, 13, (88, 5), 16), (64, 6, 15, (88, 6), 16), (70, 6, 14, (94, 5), 16), (70, 6, 7, (94, 5), 16),
    (255, 3, 13, (94, 5), 16),   # saturated scores: several keys at the maximum, others at the minimum
    (255, 0, 12, (255, 0), 12), (1, 0, 10, (3, 1), 16), (0, 5, 13, (88, 5), 16), (70, 31, 13, (88, 5), 16),
    (70, 32, 13, (88, 5), 16), (90, 6, 16, (88, 5), 16), (90, 6, 1, (88, 5), 16), (90, 6, 5, (88, 31), 13),
    (90, 6, 30, (88, 32), 29), (90, 6, 8, (88, -3), 0), (90, -2, 9, (7, 1), 15), (90, 6, 11, (88, 5), 16),
])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_parameters(ops, mult, shift, fb, av, off, D):
    c = _attn_case(fb * 100 + shift, [70, 3, 150], [18, 1, 4], 2, 1, D, 16, True, sd=40)
    _check_attn(ops, c, mult, shift, fb, av, off)


# (multiplier, shift, frac_bits): rows whose maximum saturates, rows far below 0, shifts on both sides of 9, every
# number of fraction bits
MANY_PARAMS = [(118, 8, 13), (255, 3, 13), (255, 1, 14), (255, 0, 12), (0, 5, 13), (70, 31, 13), (70, 9, 13), (90, 10, 13),
               (255, 2, 7), (30, 4, 8), (90, 6, 9), (90, 6, 10), (90, 5, 11), (120, 6, 12), (64, 6, 15), (90, 6, 16), (90, 6, 1),
               (90, 6, 6), (1, 9, 7)]


@pytest.mark.parametrize("mult,shift,fb", MANY_PARAMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("low", [False, True])
def test_tree_attention_parameters_many_rows(ops, mult, shift, fb, D, low):
    c = _attn_case(fb * 100 + shift, [70, 3, 150], [18, 40, 33], 1, 1, D, 16, True, sd=40)
    if low:  # every score far below 0
        c["q"], c["kc"] = np.abs(c["q"].astype(np.int16)).clip(1, 127).astype(np.int8), -np.abs(
            c["kc"].astype(np.int16)).clip(1, 127).astype(np.int8)
    _check_attn(ops, c, mult, shift, fb, (88, 5), 16)


def _exact_scores(xs, D):
    """A query and keys [len(xs), D] whose products are the given numbers (|x| below 4 * 127^2)."""
    xs = np.asarray(xs, np.int64)
    q = np.full(D, 127, np.int8)
    q[0] = 1
    k = np.zeros((len(xs), D), np.int64)
    rest = np.round(xs / 127).astype(np.int64)
    k[:, 0] = xs - 127 * rest
    for d in range(1, 5):
        k[:, d] = np.clip(rest, -127, 127)
        rest = rest - k[:, d]
    assert not rest.any() and np.abs(k).max() <= 127
    return q, k.astype(np.int8)


@pytest.mark.parametrize("best", [-9972, -9973, -9974, -9975])
@pytest.mark.parametrize("fb", [12, 13, 14])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [20, 2])
def test_tree_attention_other_keys_at_the_lowest_score(ops, best, fb, D, new):
    """A row's best score around -9974, every other one clamped to -32768: the clamped difference, -22795, is
    the last with a probability above 0 at 13 and 14 fraction bits, and the unclamped one has none."""
    c = _attn_case(5, [70], [new], 1, 1, D, 16, tree=False)
    q, k = _exact_scores([best, -40000], D)
    c["q"][:], c["kc"][:] = q, k[1]
    c["kc"][c["table"][0, 0], 0, 3] = k[0]
    assert np.abs(_check_attn(ops, c, 64, 6, fb, (255, 0)).cpu().numpy().astype(int)).max() > 0


@pytest.mark.parametrize("fb", range(7, 15))
@pytest.mark.parametrize("rows", [1, 9])  # the few-rows and the many-rows kernel
def test_tree_attention_every_score_difference(ops, fb, rows):
    """The short forms of the shift exponential, for every difference of a key's score and the row's best, and
    beside best and other scores past 16 bits, which are clamped: one request per pair of scores, its two keys in
    the context. The output channels weigh the two probabilities 0, 2, .. 126 to 127, so that the ones near the
    balance tell any two probabilities up to the largest ordinary one (95) apart."""
    D, page = 64, 8
    step = np.arange(65536)
    top = np.minimum(step // 2, 32767)  # best - other = step: all of 0 .. 65535
    every = np.arange(-32768, 32768)
    pairs = np.concatenate([np.stack([top, top - step], 1),                        # every difference
                            np.stack([every, np.full(65536, -40000)], 1),          # the other one clamped
                            np.stack([np.full(65536, 40000), every], 1)])          # the best one clamped
    q, k = _exact_scores(pairs.reshape(-1), D)
    x = np.clip(pairs, -32768, 32767)
    p = R.shift_exp(x, R._i16(x.max(1, keepdims=True) + 1), fb)
    v = np.stack([-2 * np.arange(D), np.full(D, 127)])
    inv = np.array([R.fisr(s, 16) for s in range(513)])[p.sum(1)]
    o = R.rounding_rshift(R._i32((p @ v) * inv[:, None]), 16)
    o = R.rounding_rshift(R._i32(o * inv[:, None]), 16)
    want = np.clip(R._i32(o * 255), -127, 127).astype(np.int8)
    i32 = lambda a: dev(np.asarray(a, np.int32))
    B = 32768
    for at in range(0, len(pairs), B):
        kc = torch.zeros(B, 1, page, D, dtype=torch.int8, device="cuda")
        vc = torch.zeros_like(kc)
        kc[:, 0, :2] = dev(k.reshape(-1, 2, D)[at:at + B])
        vc[:, 0, :2] = dev(v.astype(np.int8))
        got = ops.tree_attention_cuda(dev(q).expand(B * rows, 1, D), kc, vc, i32(np.arange(B)[:, None]), i32([2] * B),
                                      i32(np.arange(B + 1) * rows), 64, 6, fb, 255, 0,
                                      tree_mask=torch.zeros(B * rows, 1, dtype=torch.int32, device="cuda"))
        got = got.view(B, rows, D).cpu().numpy()
        assert np.array_equal(got, np.broadcast_to(want[at:at + B, None], got.shape))


@pytest.mark.parametrize("ctx,new,Hkv,G,D,page,tree", [
    ([300], [70], 2, 1, 64, 16, False),            # a chain over several blocks of rows
    ([500, 20], [30, 64], 1, 4, 64, 128, True),    # pages longer than a tile
    ([511, 513], [12, 11], 2, 1, 64, 32, True),    # around what stays in shared memory
    ([260, 700], [33, 20], 1, 2, 128, 8, True),
    ([90, 600], [20, 31], 1, 2, 128, 4, True),     # pages too short for tensor maps
    ([77, 5], [17, 40], 2, 1, 64, 2, True),
    ([3000], [24], 1, 4, 128, 64, True),           # keys split over a cluster
    ([2500, 31], [16, 1], 1, 1, 64, 16, True),
    ([0, 0], [64, 40], 1, 1, 64, 16, True),
    ([10], [300], 1, 1, 128, 16, False),
    ([1000], [200], 1, 8, 64, 16, False),
    ([40, 41, 42], [1, 1, 90], 2, 1, 64, 16, True),  # one large tree among single tokens
    ([40, 41, 42, 3, 4, 5, 6, 7], [1, 1, 50, 1, 1, 1, 1, 1], 2, 1, 64, 16, True),  # the few-rows kernel takes it
])
def test_tree_attention_many_rows(ops, ctx, new, Hkv, G, D, page, tree):
    _check_attn(ops, _attn_case(sum(ctx) + page, ctx, new, Hkv, G, D, page, tree))


@pytest.mark.parametrize("fb", [13, 14, 15])
@pytest.mark.parametrize("new", [[9, 20], [2, 3]])
def test_tree_attention_extreme_values_by_rows(ops, fb, new):
    """As test_tree_attention_extreme_values, for either kernel and wide heads."""
    for D in (64, 128):
        c = _attn_case(3, [40, 5], new, 1, 1, D, 16)
        for qv, kv, vv in ((-128, -128, -128), (127, -128, 127), (-128, 127, -128)):
            c["q"][:], c["kc"][:], c["vc"][:] = qv, kv, vv
            _check_attn(ops, c, 255, 4, fb, (255, 2))
        c["q"][:] = 127
        c["kc"][::2], c["kc"][1::2] = 127, -128
        for shift in (0, 2, 4, 9):
            _check_attn(ops, c, 255, shift, fb, (88, 5))


def test_tree_attention_holes_many_rows(ops):
    for D, page in ((64, 16), (128, 64), (64, 128), (64, 4)):
        c = _attn_case(9, [260, 140, 300], [25, 36, 17], 2, 1, D, page)
        c["table"][0, 1], c["table"][1, 0], c["table"][2, 2] = -1, 10 ** 6, -7
        c["ctx"][1] = 5000
        _check_attn(ops, c)


def test_tree_attention_rows_that_see_nothing_many_rows(ops):
    c = _attn_case(11, [0, 0, 20], [39, 20, 39], 2, 2, 64, 8, empty_rows=True)
    assert _check_attn(ops, c)[1].count_nonzero() == 0


@pytest.mark.parametrize("fb", [13, 15])
def test_tree_attention_extreme_values(ops, fb):
    """-128 everywhere, alternating extremes, and negative scores only."""
    c = _attn_case(3, [40, 5], [9, 20], 2, 1, 64, 16)
    for qv, kv, vv in ((-128, -128, -128), (127, -128, 127), (-128, 127, -128)):
        c["q"][:], c["kc"][:], c["vc"][:] = qv, kv, vv
        _check_attn(ops, c, 255, 4, fb, (255, 2))
    c["q"][:] = 127
    c["kc"][::2], c["kc"][1::2] = 127, -128  # best and worst key at once: the difference leaves 16 bits
    _check_attn(ops, c, 255, 0, fb, (88, 5))


def test_tree_attention_rows_that_see_nothing(ops):
    c = _attn_case(11, [0, 0, 20], [9, 1, 9], 2, 2, 64, 8, empty_rows=True)
    got = _check_attn(ops, c)
    assert got[1].count_nonzero() == 0  # empty mask, no context


@pytest.mark.parametrize("order", ["prhd", "hprd"])
def test_tree_attention_cache_orders(ops, order):
    _check_attn(ops, _attn_case(5, [77, 400], [6, 21], 4, 1, 64, 16, order=order))


def test_tree_attention_strided_query_and_output(ops):
    c = _attn_case(6, [50, 9], [11, 30], 4, 1, 64, 16)
    N, H, D = c["q"].shape
    want = _check_attn(ops, c)
    qkv = torch.zeros(N, 3 * H * D, dtype=torch.int8, device="cuda")
    qkv[:, H * D:2 * H * D] = dev(c["q"]).view(N, H * D)
    canvas = torch.full((N + 2, H * D + 32), 55, dtype=torch.int8, device="cuda")
    got = ops.tree_attention_cuda(qkv[:, H * D:2 * H * D].view(N, H, D), dev(c["kc"]), dev(c["vc"]), dev(c["table"]),
                                  dev(c["ctx"]), dev(c["starts"]), 70, 6, 13, 88, 5, tree_mask=dev(c["mask"]),
                                  out=canvas[1:-1, 16:-16])
    assert torch.equal(got, want)
    edge = canvas.clone()
    edge[1:-1, 16:-16] = 55
    assert bool((edge == 55).all())  # nothing outside the output was written


def test_tree_attention_padding_rows_and_missing_pages(ops):
    """Rows past starts[B] give 0; a page of -1 or past the cache hides its keys; a context longer than the
    block table is cut to it."""
    c = _attn_case(8, [70, 40, 100], [5, 6, 7], 2, 1, 64, 16)
    c["table"][0, 2], c["table"][1, 0] = -1, 10 ** 6
    c["ctx"][2] = 500
    c["q"] = np.concatenate([c["q"], c["q"][:9]])
    c["mask"] = np.concatenate([c["mask"], c["mask"][:9]])
    got = _check_attn(ops, c)
    assert got[18:].count_nonzero() == 0


def test_tree_attention_no_requests(ops):
    """Every row is padding."""
    z = lambda *s, dtype=torch.int8: torch.zeros(*s, dtype=dtype, device="cuda")
    out = torch.full((5, 128), 7, dtype=torch.int8, device="cuda")
    ops.tree_attention_cuda(z(5, 2, 64), z(3, 2, 16, 64), z(3, 2, 16, 64), z(0, 4, dtype=torch.int32), z(0, dtype=torch.int32),
                            z(1, dtype=torch.int32), 70, 6, 13, 88, 5, out=out)
    assert out.count_nonzero() == 0


def test_tree_attention_wide_block_table_and_many_requests(ops):
    rng = np.random.default_rng(1)
    ctx, new = rng.integers(0, 90, 300).tolist(), rng.integers(0, 4, 300).tolist()
    _check_attn(ops, _attn_case(1, ctx, new, 1, 1, 64, 16, tree=False, extra_width=700))


def test_tree_attention_long_context(ops):
    """More keys than a block's shared memory holds, one row and sixteen."""
    c = _attn_case(2, [9001, 20000], [1, 1], 1, 1, 64, 16, tree=False)
    _check_attn(ops, c, 100, 7)
    c = _attn_case(2, [12007], [8], 1, 2, 128, 32, tree=True)
    _check_attn(ops, c, 70, 7)


def test_tree_attention_sums_wrap_and_offsets_past_32_bits(ops):
    """70,000 keys at the largest probability and value: the P.V sum wraps in 32 bits as the definition says;
    the pages lie beyond 2^31 bytes of the cache."""
    P, page, D = 40000, 1024, 64
    kc = torch.zeros(P, 1, page, D, dtype=torch.int8, device="cuda")  # 2.6 GB
    vc = kc
    pages = np.arange(P - 69, P, dtype=np.int32)[None]
    kc[P - 69:] = -128
    ctx, starts = np.asarray([69 * 1024 - 1], np.int32), np.asarray([0, 1], np.int32)
    q = np.zeros((1, 1, D), np.int8)
    got = ops.tree_attention_cuda(dev(q), kc, vc, dev(pages), dev(ctx), dev(starts), 70, 6, 15, 88, 5)
    small = np.full((69, 1, page, D), -128, np.int8)
    want = R.tree_attention(q, small, small, np.arange(69, dtype=np.int32)[None], ctx, starts, 70, 6, 15, 88, 5)
    assert np.array_equal(got.cpu().numpy(), want)


def test_tree_attention_matches_dense_attention(ops):
    """A batch of equal chains gives the bytes of the dense causal attention."""
    rng = np.random.default_rng(4)
    B, H, T, L, D, page = 3, 4, 5, 96, 64, 16
    q, k, v = (dev(rng.integers(-60, 61, (B, n, H * D), dtype=np.int8)) for n in (T, L, L))
    dense = ops.attention_cuda(q, k, v, H, 70, 7, 13, 88, 5, mask_mode=1)
    pages = lambda x: x.view(B, L // page, page, H, D).permute(0, 1, 3, 2, 4).reshape(-1, H, page, D).contiguous()
    i = lambda *x: dev(np.asarray(x, np.int32))
    table = torch.arange(B * L // page, dtype=torch.int32, device="cuda").view(B, -1)
    got = ops.tree_attention_cuda(q.view(B * T, H, D), pages(k), pages(v), table, i(*[L - T] * B), i(0, T, 2 * T, 3 * T),
                                  70, 7, 13, 88, 5)
    assert torch.equal(got.view(B, T, H * D), dense)


def test_tree_attention_on_another_stream_and_in_a_graph(ops):
    c = _attn_case(12, [300, 17], [9, 3], 2, 1, 64, 16)
    args = [dev(c[n]) for n in ("q", "kc", "vc", "table", "ctx", "starts")]
    mask = dev(c["mask"])
    want = ops.tree_attention_cuda(*args, 70, 6, 13, 88, 5, tree_mask=mask)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.tree_attention_cuda(*args, 70, 6, 13, 88, 5, tree_mask=mask)
    st.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(want)
    with torch.cuda.graph(g):
        ops.tree_attention_cuda(*args, 70, 6, 13, 88, 5, tree_mask=mask, out=out)
    args[4].sub_(2)  # shorter contexts, read on the device
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.tree_attention_cuda(*args, 70, 6, 13, 88, 5, tree_mask=mask))
    assert not torch.equal(out, want)


def test_tree_attention_refusals(ops):
    z = lambda *s, dtype=torch.int8: torch.zeros(*s, dtype=dtype, device="cuda")
    i = lambda *s: z(*s, dtype=torch.int32)
    kc = z(3, 2, 16, 64)
    call = lambda q=z(4, 2, 64), kc=kc, t=i(1, 3), c=i(1), s=i(2), fb=13, off=16, **kw: ops.tree_attention_cuda(
        q, kc, kc, t, c, s, 70, 6, fb, 88, 5, rsqrt_offset=off, **kw)
    call()
    for match, kw in (("divide", dict(q=z(4, 3, 64))), ("64 or 128", dict(q=z(4, 2, 32), kc=z(3, 2, 16, 32))),
                      ("dimension mismatch", dict(q=z(4, 2, 128))), ("frac_bits", dict(fb=31)),
                      ("rsqrt_offset", dict(off=30)), ("power of two", dict(kc=z(3, 2, 12, 64))),
                      ("starts", dict(s=i(3))), ("context_lens", dict(c=i(2))), ("tree_mask", dict(tree_mask=i(3, 1))),
                      ("block_table", dict(t=i(3))), ("16-byte", dict(q=z(4, 2, 72)[:, :, 8:])),
                      ("out must", dict(out=z(4, 64))), ("2\\^23", dict(t=i(1, 600000))),
                      ("int8", dict(q=z(4, 2, 64, dtype=torch.int16)))):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    assert call(q=z(0, 2, 64)).shape == (0, 128)


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def _lp_tol(V, x, scale):
    """A sum of V positive terms over at least 128 threads is V/128 additions in a row and a tree of at most
    16 more, each within 2^-24 of its result; exp and log are within 2 ulp, and every logit, the maximum and
    the differences are rounded once; terms more than 100 below the maximum vanish, so the logits that count
    are no larger than the row's maximum plus 100. The entropy weights this by the mean distance from the maximum, at most
    log V plus the entropy's own size. -> [N, 1]"""
    some = np.isfinite(x).any(1, keepdims=True)
    top = np.where(some, np.where(np.isfinite(x), x, -np.inf).max(1, keepdims=True), 0.0) * scale
    low = np.where(some, np.where(np.isfinite(x), x, np.inf).min(1, keepdims=True), 0.0) * scale
    big = np.abs(top) + np.minimum(100.0, top - low)
    return 2.0 ** -24 * (V / 128 + 32 + 8 * big) * (1 + np.log(V))


def _check_lp(ops, x, targets, top, scale=1.0, bits=None):
    V = x.shape[1]
    sup = None
    if bits is not None:
        sup = ((bits.cpu().numpy().astype(np.int64)[:, None] >> np.arange(32)) & 1).reshape(-1)[:V].astype(bool)
    x64 = x.double().cpu().numpy()
    want = R.token_logprobs(x64, targets, top, scale, sup)
    got = ops.token_logprobs_cuda(x, dev(targets) if targets.shape[1] else None, top, scale, bits)
    assert np.array_equal(got[2].cpu().numpy(), want[2])
    tol = _lp_tol(V, x64, scale)
    for g, w in ((got[0], want[0]), (got[1][:, None], want[1][:, None]), (got[3], want[3])):
        g = g.double().cpu().numpy()
        fine = np.isfinite(w)
        assert np.array_equal(g[~fine], w[~fine], equal_nan=True)
        off = np.abs(np.where(fine, g, 0) - np.where(fine, w, 0))
        assert (off <= tol + 2e-6 * np.abs(np.where(fine, w, 0))).all(), (off.max(), tol.max())
    return got


def _logits(rng, kind, N, V, ld=None, sd=3.0):
    ld = ld or V
    if kind == "int8":
        return dev(np.clip(np.round(rng.normal(0, 8 * sd, (N, ld))), -128, 127).astype(np.int8))[:, :V]
    return dev(rng.normal(0, sd, (N, ld)).astype(np.float32)).to(getattr(torch, kind))[:, :V]


KINDS = ["int8", "float16", "bfloat16", "float32"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,V,ld,C,top", [(1, 1, None, 1, 1), (2, 2, None, 1, 2), (3, 31, 40, 2, 5), (1, 33, None, 0, 32),
                                          (7, 257, 259, 1, 1), (5, 4099, 4103, 3, 20), (2, 51865, 51872, 1, 5),
                                          (150, 2050, None, 1, 0), (1, 130001, 130004, 2, 32), (300, 700, 701, 1, 3)])
def test_logprobs(ops, kind, N, V, ld, C, top):
    rng = np.random.default_rng(V + N)
    t = rng.integers(0, V, (N, C))
    if C > 1:
        t[::2, -1] = -1
    _check_lp(ops, _logits(rng, kind, N, V, ld), t, min(top, V), 0.125 if kind == "int8" else 1.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [5, 64, 5000, 51866])
def test_logprobs_suppressed(ops, kind, V):
    rng = np.random.default_rng(V)
    x = _logits(rng, kind, 4, V)
    bits = rng.integers(-2 ** 31, 2 ** 31, (V + 31) // 32).astype(np.int32)
    _check_lp(ops, x, rng.integers(0, V, (4, 3)), min(V, 8), 0.3, dev(bits))
    nearly = np.full((V + 31) // 32, -1, np.int32)
    nearly[1 % len(nearly)] ^= 1 << 3  # one token left
    _check_lp(ops, x, rng.integers(0, V, (4, 3)), min(V, 8), 1.0, dev(nearly).view(torch.uint32))
    got = _check_lp(ops, x, rng.integers(0, V, (4, 3)), min(V, 8), 1.0, dev(np.full_like(nearly, -1)))
    assert bool((got[0] == -np.inf).all()) and bool((got[2] == -1).all())


@pytest.mark.parametrize("kind", KINDS)
def test_logprobs_equal_logits_go_by_id(ops, kind):
    rng = np.random.default_rng(2)
    for V in (40, 3000, 52001):
        x = torch.zeros(3, V, device="cuda")
        x[1] = dev(rng.integers(-1, 2, V).astype(np.float32))
        x[2, V // 2:] = 5
        _check_lp(ops, x.to(getattr(torch, kind)), rng.integers(0, V, (3, 1)), 32)


def test_logprobs_signed_zeros_are_equal(ops):
    for kind in (torch.float16, torch.bfloat16, torch.float32):
        x = torch.full((1, 4000), -1.0, device="cuda").to(kind)
        x[0, 100:200] = 0.0
        x[0, 50:100] = -0.0
        assert ops.token_logprobs_cuda(x, top=32)[2].tolist() == [list(range(50, 82))]


def test_logprobs_largest_first_and_last(ops):
    for V in (4097, 51865):
        for at in (0, V - 1, V // 2):
            x = torch.full((2, V), -100, dtype=torch.int8, device="cuda")
            x[:, at] = 100
            _check_lp(ops, x, np.full((2, 1), at), 3, 0.25)


@pytest.mark.parametrize("kind", ["float16", "bfloat16", "float32"])
def test_logprobs_infinities_and_nan(ops, kind):
    rng = np.random.default_rng(5)
    for V in (70, 6001):
        x = _logits(rng, kind, 8, V).clone()
        x[0] = -np.inf
        x[1, 7:] = -np.inf
        x[2, 3] = np.inf
        x[3, V - 1] = np.nan
        x[4] = torch.finfo(x.dtype).min  # a mask of the type's lowest value: an ordinary, equal logit
        x[5, 1:] = torch.finfo(x.dtype).min
        t = rng.integers(0, V, (8, 2))
        t[1] = 9
        t[6] = [V, -5]
        got = _check_lp(ops, x, t, 10)
        assert got[2][0].tolist() == [-1] * 10 and got[1][0].item() == 0.0
        assert got[2][1].tolist()[7:] == [-1] * 3
        bits = torch.zeros((V + 31) // 32, dtype=torch.int32, device="cuda")
        bits[0] = 8  # the +inf of row 2 is suppressed, and so are the bits past V of no concern
        got = _check_lp(ops, x, t, 10, 1.0, bits)
        assert bool(torch.isfinite(got[1][2]))


def test_logprobs_unaligned_rows(ops):
    rng = np.random.default_rng(6)
    for kind in KINDS:
        x = _logits(rng, kind, 5, 3001, 3003)[:, 1:]
        _check_lp(ops, x, rng.integers(0, 3000, (5, 1)), 4, 0.5)


def test_logprobs_scale_keeps_the_order_of_the_logits(ops):
    """Logits that differ in their last bit keep their order however they are scaled."""
    base = np.float32(1.0)
    x = np.full((1, 2000), -3.0, np.float32)
    for i in range(10):
        x[0, 100 + i] = base
        base = np.nextafter(base, np.float32(2.0))
    ids = ops.token_logprobs_cuda(dev(x), top=10, scale=0.3)[2]
    assert ids.tolist() == [list(range(109, 99, -1))]


def test_logprobs_rows_past_2_to_31_elements(ops):
    N, V = 42000, 51872  # 2.2e9 logits
    x = torch.full((N, V), -90, dtype=torch.int8, device="cuda")
    x[-1, 17] = 33
    x[-1, 51871] = 34
    lp, ent, ids, top = ops.token_logprobs_cuda(x, top=2, scale=1.0)
    assert ids[-1].tolist() == [51871, 17] and ids[0].tolist() == [0, 1]
    np.testing.assert_allclose(top[-1].cpu().numpy(), [-np.log1p(np.exp(-1.0)), -1 - np.log1p(np.exp(-1.0))], rtol=1e-5)


def test_logprobs_refusals(ops):
    x = torch.zeros(3, 50, device="cuda")
    for match, a, kw in (("top", x, dict(top=33)), ("top", x[:, :4], dict(top=5)), ("scale", x, dict(scale=0.0)),
                         ("scale", x, dict(scale=float("nan"))), ("float32", x.double(), {}),
                         ("contiguous rows", x.t(), {}), ("targets", x, dict(targets=torch.zeros(3, 1, device="cuda"))),
                         ("suppress_bits", x, dict(suppress_bits=torch.zeros(1, dtype=torch.int32, device="cuda"))),
                         ("logits must be", x[0], {})):
        with pytest.raises(RuntimeError, match=match):
            ops.token_logprobs_cuda(a, **kw)
    lp, ent, ids, top = ops.token_logprobs_cuda(x[:0], top=2)
    assert lp.shape == (0, 0) and ent.shape == (0,) and ids.shape == top.shape == (0, 2)


def test_numbers_out_of_range_are_refused_like_other_arguments(ops):
    z = lambda *s, dtype=torch.int8: torch.zeros(*s, dtype=dtype, device="cuda")
    i = lambda *s: z(*s, dtype=torch.int32)
    kc = z(3, 2, 16, 64)
    good = [70, 6, 13, 88, 5]
    for at, bad in ((0, 256), (0, -1), (1, 128), (2, 2 ** 31), (3, 300), (4, -129)):
        args = list(good)
        args[at] = bad
        with pytest.raises(RuntimeError, match="iw_tree_attention"):
            ops.tree_attention_cuda(z(4, 2, 64), kc, kc, i(1, 3), i(1), i(2), *args)
    with pytest.raises(RuntimeError, match="iw_tree_attention"):
        ops.tree_attention_cuda(z(4, 2, 64), kc, kc, i(1, 3), i(1), i(2), *good, rsqrt_offset=2 ** 40)
    for scale in (1e39, "1"):
        with pytest.raises(RuntimeError, match="iw_token_logprobs"):
            ops.token_logprobs_cuda(z(3, 50), scale=scale)
    with pytest.raises(RuntimeError, match="iw_paged_plan"):
        ops.paged_plan_cuda(i(2), i(2), i(2, 4), i(1), i(1), 16.0, 2)


def test_outputs_that_overlap_are_refused(ops):
    z = lambda *s, dtype=torch.int8: torch.zeros(*s, dtype=dtype, device="cuda")
    i = lambda *s: z(*s, dtype=torch.int32)
    kc, k, slots = z(3, 2, 16, 64), z(4, 2, 64), z(4, dtype=torch.int64)
    for cache in (kc[:1].expand(3, -1, -1, -1), kc[:, :1].expand(-1, 2, -1, -1), kc[:, :, :1].expand(-1, -1, 16, -1),
                  kc.view(-1).as_strided((3, 2, 16, 64), (1024, 1024, 64, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.paged_kv_write_cuda(k, k, slots, cache, cache)
    args = (k, kc, kc, i(1, 3), i(1), i(2), 70, 6, 13, 88, 5)
    for out in (z(1, 128).expand(4, -1), z(1024).as_strided((4, 128), (64, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.tree_attention_cuda(*args, out=out)
    # one page, head or row: its stride says nothing; caches that lie between one another's rows are apart
    both = z(3, 2, 2, 16, 64)
    ops.paged_kv_write_cuda(k, k, slots, both[:, 0], both[:, 1])
    for cache in (kc[:1], kc[:, :, :1]):
        ops.paged_kv_write_cuda(k, k, slots, cache, cache)
    ops.paged_kv_write_cuda(k[:, :1], k[:, :1], slots, kc[:, :1], kc[:, :1])
    ops.tree_attention_cuda(k[:1], *args[1:], out=z(1, 128).as_strided((1, 128), (0, 1)))


@pytest.mark.parametrize("kind", ["float16", "bfloat16", "float32"])
def test_logprobs_gradients_are_refused(ops, kind):
    """Logits that ask for a gradient give the same scores, and an error where it would be lost."""
    x = _logits(np.random.default_rng(3), kind, 4, 300).clone()
    t = torch.tensor([[1], [2], [3], [-1]], device="cuda")
    want = ops.token_logprobs_cuda(x, t, 3)
    x.requires_grad_()
    got = ops.token_logprobs_cuda(x, t, 3)
    assert all(torch.equal(g.detach(), w) for g, w in zip(got, want))
    for g in (got[0], got[1], got[3]):
        with pytest.raises(RuntimeError, match="no gradient"):
            g.sum().backward(retain_graph=True)
    assert not got[2].requires_grad
    with torch.no_grad():
        assert not any(g.requires_grad for g in ops.token_logprobs_cuda(x, t, 3))


# Small batches leave each block one row at a time; with enough (request, key head) pairs the few-rows kernel takes
# eight rows at a time, by 1, 2 or 4 warps a pair and by clusters (the block table's width decides)
def _many_pairs(seed, B, most, G, width_keys, page, long=()):
    """Contexts, new-token counts (at most 8 / G on average) and the spare columns that make the block table
    `width_keys` keys wide; `long` requests come first."""
    rng = np.random.default_rng(seed)
    new = rng.integers(1, 8 // G + 1, B)
    ctx = rng.integers(0, most + 1, B)
    ctx[1::7], new[2::9] = 0, 0
    for i, (c, n) in enumerate(long):
        ctx[i], new[i] = c, n
    cols = -(-int((ctx + new).max()) // page)
    return ctx.tolist(), new.tolist(), max(width_keys // page - cols, 0)


@pytest.mark.parametrize("B,Hkv,G,most,width_keys,long", [
    (150, 4, 1, 50, 64, ()),                          # a warp per pair
    (76, 8, 1, 110, 128, ()),                         # two
    (40, 4, 2, 200, 256, ()),                         # four
    (40, 4, 1, 60, 1024, ((900, 5), (1010, 7))),      # clusters
])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 4])             # TMA; pages too short for it
@pytest.mark.parametrize("tree,holes", [(True, False), (False, True), (True, True)])
def test_tree_attention_eight_rows_at_a_time(ops, B, Hkv, G, most, width_keys, long, D, page, tree, holes):
    ctx, new, spare = _many_pairs(B + D + page, B, most, G, width_keys, page, long)
    c = _attn_case(B + page, ctx, new, Hkv, G, D, page, tree, extra_width=spare, empty_rows=holes)
    if holes:
        rng = np.random.default_rng(B)
        at = rng.integers(0, 8, (c["table"].shape[0], 2)) % np.maximum(1, -(-c["ctx"][:, None] // page))
        c["table"][np.arange(0, B, 3), at[::3, 0]] = -1
        c["table"][np.arange(0, B, 5), at[::5, 1]] = 10 ** 6
    _check_attn(ops, c)


@pytest.mark.parametrize("mult,shift,fb,av,off", [(255, 3, 13, (94, 5), 16), (255, 0, 12, (255, 0), 12), (64, 6, 15, (88, 6), 16),
                                                  (0, 5, 13, (88, 5), 16), (90, 6, 1, (88, 5), 16), (90, 6, 30, (88, 32), 29),
                                                  (255, 2, 7, (88, 5), 16), (64, 6, 14, (255, 0), 16)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("low", [False, True])
def test_tree_attention_parameters_eight_rows_at_a_time(ops, mult, shift, fb, av, off, D, low):
    ctx, new, spare = _many_pairs(fb + D, 150, 50, 1, 64, 16)
    c = _attn_case(fb, ctx, new, 4, 1, D, 16, True, sd=60, extra_width=spare)
    if low:  # every score far below 0
        c["q"], c["kc"] = np.abs(c["q"].astype(np.int16)).clip(1, 127).astype(np.int8), -np.abs(
            c["kc"].astype(np.int16)).clip(1, 127).astype(np.int8)
    _check_attn(ops, c, mult, shift, fb, av, off)


@pytest.mark.parametrize("D,page,G,tree", [(64, 16, 1, True), (128, 16, 1, False), (64, 4, 2, True), (128, 64, 2, True), (64, 64, 1, False)])
@pytest.mark.parametrize("holes", [False, True])
def test_tree_attention_more_scores_than_a_warp_keeps(ops, D, page, G, tree, holes):
    """Requests of 20000 keys and several rows among short ones: their scores do not fit shared memory and are
    computed again from K in global memory in the second pass."""
    ctx, new, spare = _many_pairs(D + page, 20, 300, G, 65536, page, ((20000, 8), (19000, 11)))
    c = _attn_case(D * G + page, ctx, new, 1, G, D, page, tree, extra_width=spare)
    if holes:
        c["table"][0, 7], c["table"][0, 200], c["table"][1, 1] = -1, 10 ** 6, -1
    _check_attn(ops, c, 70, 7)


def test_no_wait_ran_out(ops):
    from i_whisper_b200 import _lib
    assert _lib.device_status(clear=True) == 0
