"""The plain implementations that the GPU tests of the paged operators compare
with, checked on the CPU: the tree attention against the oracle's dense
attention stages, the log probabilities against torch, the plan by its own
rules. And the refusals of the C entry points, which need no GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_reference as R
from oracle import oracle as O

from i_whisper_b200.build import build

build()  # the library is compiled in-tree (a no-op when up to date)
from i_whisper_b200 import _lib  # noqa: E402


@pytest.fixture(scope="module")
def L():
    return O.lib("port")


@pytest.mark.parametrize("mult,shift,fb,av,off", [(70, 6, 13, (88, 5), 16), (118, 8, 7, (94, 5), 16),
                                                  (255, 0, 12, (255, 0), 13), (90, 3, 10, (3, 1), 16)])
def test_tree_attention_reference_is_the_oracles(L, mult, shift, fb, av, off):
    rng = np.random.default_rng(fb)
    H, T, Lk, D, page = 3, 6, 48, 64, 16
    q, k, v = (rng.integers(-90, 91, (1, H, n, D), dtype=np.int8) for n in (T, Lk, Lk))
    mask = np.arange(Lk)[None] > Lk - T + np.arange(T)[:, None]
    qk, rm = L.qk_requant_rowmax(q, k, mask, mult, shift)
    p, rs = L.shift_exp(qk, rm, mask, fb)
    want = L.pv_norm_requant(p, np.ascontiguousarray(v.transpose(0, 1, 3, 2)), rs, *av, off)
    pages = lambda x: x[0].reshape(H, Lk // page, page, D).transpose(1, 0, 2, 3)
    table, ctx, starts = np.arange(Lk // page, dtype=np.int32)[None], [Lk - T], [0, T]
    args = (q[0].transpose(1, 0, 2), pages(k), pages(v), table, ctx, starts, mult, shift, fb, *av, off)
    assert np.array_equal(R.tree_attention(*args), np.asarray(want)[0])
    bits = (((1 << (np.arange(T) + 1)) - 1)[:, None]).astype(np.int32)  # the chain as a tree mask
    assert np.array_equal(R.tree_attention(*args, mask=bits), np.asarray(want)[0])


def test_logprobs_reference_is_torchs():
    rng = np.random.default_rng(0)
    x = rng.normal(0, 3, (4, 300))
    t = rng.integers(0, 300, (4, 2))
    lp, ent, ids, top = R.token_logprobs(x, t, 6, 0.7)
    ref = torch.log_softmax(torch.from_numpy(x) * 0.7, 1)
    assert np.allclose(lp, ref.gather(1, torch.from_numpy(t)), atol=1e-12)
    assert np.allclose(ent, -(ref.exp() * ref).sum(1), atol=1e-12)
    assert np.array_equal(ids, ref.topk(6, 1).indices) and np.allclose(top, ref.topk(6, 1).values, atol=1e-12)


def test_plan_reference_by_hand():
    p = R.paged_plan([3, 0, 16], [2, 0, 17], np.full((3, 4), 9, np.int32), np.array([40, 41, 42], np.int32), 1, 16, 20)
    assert p["starts"].tolist() == [0, 2, 2, 19] and p["free_head"] == 3 and p["status"] == 0
    assert p["slots"][:4].tolist() == [147, 148, 41 * 16, 41 * 16 + 1] and p["slots"][18:].tolist() == [42 * 16, -1]
    assert p["table"][2].tolist() == [9, 41, 42, 9] and p["table"][:2].tolist() == [[9] * 4] * 2
    assert p["position"][:4].tolist() == [3, 4, 16, 17] and p["request"][18:].tolist() == [2, -1]


FAKE = 0x1000  # a 16-byte aligned placeholder address


def _reject(entry, cls, good, cases):
    for changes, needle in cases:
        d = cls(**{**good, **changes})
        assert getattr(_lib.LIB, entry)(C.byref(d), None) == _lib.IW_EINVAL, changes
        assert needle in _lib.last_error(), (changes, _lib.last_error())
    assert getattr(_lib.LIB, entry)(None, None) == _lib.IW_EINVAL


def test_paged_plan_refusals():
    good = {n: FAKE for n in ("context_lens", "new_lens", "block_table", "free_pages", "free_head", "slots", "request",
                              "position", "starts", "status")}
    good.update(B=2, table_ld=4, table_width=4, n_free=9, page_size=16, max_tokens=5, free_head_out=FAKE + 64)
    _reject("iw_paged_plan", _lib.PagedPlanDesc, good, [
        (dict(B=0), "request count"), (dict(B=16385), "request count"), (dict(table_ld=3), "invalid shape"),
        (dict(max_tokens=-1), "invalid shape"), (dict(n_free=-1), "invalid shape"), (dict(page_size=12), "power of two"),
        (dict(page_size=0), "power of two"), (dict(page_size=1 << 21), "power of two"), (dict(slots=None), "null array"),
        (dict(parents=FAKE), "max_new"), (dict(parents=FAKE, max_new=4), "null array"),
        (dict(free_head_out=FAKE), "free_head_out")])


def test_paged_kv_write_refusals():
    good = [FAKE, 256, 64, FAKE, 256, 64, FAKE, FAKE, FAKE, 4096, 1024, 64, 8, 16, 3, 4, 64, None]
    for at, value, needle in ((1, 250, "16-byte"), (0, FAKE + 8, "16-byte"), (13, 24, "power of two"), (14, -1, "shape"),
                              (16, 8, "shape"), (16, 72, "16-byte"), (6, None, "null"), (15, 0, "shape")):
        args = list(good)
        args[at] = value
        with pytest.raises(RuntimeError, match=needle):
            _lib.call("iw_paged_kv_write", *args)
    args = list(good)
    args[14] = 0
    _lib.call("iw_paged_kv_write", *args)  # no rows: nothing to do


def test_tree_attention_refusals():
    good = dict(q=FAKE, ldq=256, q_hs=64, y=FAKE, ldy=256, k_cache=FAKE, v_cache=FAKE, page_stride=4096, head_stride=1024,
                row_stride=64, n_pages=8, page_size=16, block_table=FAKE, table_ld=4, table_width=4, context_lens=FAKE,
                starts=FAKE, B=2, N=5, H=4, Hkv=4, D=64, frac_bits=13, rsqrt_offset=16)
    _reject("iw_tree_attention", _lib.TreeAttnDesc, good, [
        (dict(B=-1), "invalid shape"), (dict(B=65536), "invalid shape"), (dict(N=-1), "invalid shape"),
        (dict(table_ld=3), "invalid shape"), (dict(Hkv=3), "multiple"), (dict(D=96), "64 or 128"),
        (dict(page_size=24), "power of two"), (dict(table_ld=1 << 20, table_width=1 << 20), "2^23"),
        (dict(frac_bits=0), "frac_bits"), (dict(rsqrt_offset=-1), "rsqrt_offset"), (dict(q=None), "null array"),
        (dict(tree_mask=FAKE), "null array"), (dict(row_stride=72), "16-byte"), (dict(y=FAKE + 4), "16-byte")])
    assert _lib.LIB.iw_tree_attention(C.byref(_lib.TreeAttnDesc(**{**good, "N": 0})), None) == _lib.IW_OK


def test_token_logprobs_refusals():
    good = dict(logits=FAKE, ld=100, dtype=0, N=3, V=100, scale=1.0, entropy=FAKE)
    _reject("iw_token_logprobs", _lib.TokenLogprobsDesc, good, [
        (dict(V=0), "invalid shape"), (dict(ld=99), "invalid shape"), (dict(C=-1), "invalid shape"), (dict(dtype=4), "dtype"),
        (dict(top=33), "top"), (dict(top=5, V=4), "top"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
        (dict(C=1), "null array"), (dict(top=1), "null array"), (dict(dtype=3, logits=FAKE + 2), "aligned")])
    assert _lib.LIB.iw_token_logprobs(C.byref(_lib.TokenLogprobsDesc(**{**good, "N": 0})), None) == _lib.IW_OK


def test_outputs_that_overlap_are_refused():
    """Rows of one output that share memory would be written by several blocks at once."""
    attn = dict(q=FAKE, ldq=256, q_hs=64, y=FAKE, ldy=256, k_cache=FAKE, v_cache=FAKE, page_stride=4096, head_stride=1024,
                row_stride=64, n_pages=8, page_size=16, block_table=FAKE, table_ld=4, table_width=4, context_lens=FAKE,
                starts=FAKE, B=2, N=5, H=4, Hkv=4, D=64, frac_bits=13, rsqrt_offset=16)
    _reject("iw_tree_attention", _lib.TreeAttnDesc, attn, [(dict(ldy=n), "overlap") for n in (0, 64, 240)])
    # page_stride, head_stride, row_stride of [8, 4, 16, 64] caches
    for strides in ((0, 1024, 64), (4096, 0, 64), (4096, 1024, 0), (4096, 1024, 48), (4080, 1024, 64), (4096, 1008, 64),
                    (64, 512, 512), (2 ** 62, 1024, 32), (1024, 4096, 64)):
        args = [FAKE, 256, 64, FAKE, 256, 64, FAKE, FAKE, FAKE, *strides, 8, 16, 3, 4, 64, None]
        with pytest.raises(RuntimeError, match="overlap"):
            _lib.call("iw_paged_kv_write", *args)
