"""Torch-tensor operators of paged, tree-drafted decoding.

These have no counterpart among the reference's operators: they serve ragged
batches of requests whose K/V lie in pages of a shared INT8 cache, and drafted
token trees that are verified in one pass. Layouts and rules are those of the
``iw_paged_plan`` / ``iw_paged_kv_write`` / ``iw_tree_attention`` /
``iw_token_logprobs`` entries of include/iwhisper_b200.h. All work is queued on
the current stream and nothing is read on the host; arguments are checked
like the other operators' (``RuntimeError``). ``ops`` exports them too, and
``tree.TreeDecoder`` runs them together.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib

# the current stream's handle and the current device without the checks and objects
# of torch.cuda around them (a CUDA tensor is at hand, so CUDA is initialised)
if hasattr(torch._C, "_cuda_getCurrentRawStream") and hasattr(torch._C, "_cuda_getDevice"):
    _raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
else:
    _current_device = torch.cuda.current_device

    def _raw_stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _scalar(t, name: str) -> int:
    if isinstance(t, torch.Tensor):
        if t.numel() != 1:
            raise RuntimeError(f"{name} must be a scalar tensor")
        return int(t.item())
    return int(t)


class PagedPlan(NamedTuple):
    """One step's plan (``paged_plan_cuda``)."""
    slots: torch.Tensor                # [max_tokens] int64 cache slot of each new token, -1: none
    request: torch.Tensor              # [max_tokens] int32 request of each row, -1: padding
    position: torch.Tensor             # [max_tokens] int32 text position: context length + depth in the tree
    starts: torch.Tensor               # [B + 1] int32 first row of each request
    free_head: torch.Tensor            # [1] int32 the free list's head after this step
    status: torch.Tensor               # [1] int32 _lib.PLAN_* bits, 0: everything has its place
    tree_mask: Optional[torch.Tensor]  # [max_tokens, ceil(max_new/32)] int32 ancestor-or-self bits


# The descriptors of these calls as packed bytes, laid out like the C structs: a
# few times cheaper than filling a ctypes.Structure, and these calls are a step's
# host time.
_PLAN_DESC = struct.Struct("@PPqPqqPqPqqPqPPPPPPP")
_ATTN_DESC = struct.Struct("@PqqPqPPqqqqqPqqPPPqqqqqqBbiBbi0q")
_LOGP_DESC = struct.Struct("@PqiqqfPPqqPPPP")
assert (_PLAN_DESC.size, _ATTN_DESC.size, _LOGP_DESC.size) == tuple(
    ctypes.sizeof(d) for d in (_lib.PagedPlanDesc, _lib.TreeAttnDesc, _lib.TokenLogprobsDesc))


def _call(name: str, desc: struct.Struct, device: int, *args) -> None:
    try:
        packed = desc.pack(*args)
    except (struct.error, OverflowError) as e:  # a number that its C field does not hold
        raise RuntimeError(f"{name}: argument out of range: {e}") from None
    _lib.call(name, packed, _raw_stream(device))


def _chk1(t, name: str, dtype: torch.dtype, n: int, device: int):
    """A contiguous CUDA tensor [n] of `dtype` on CUDA device `device`."""
    if t.dtype is not dtype or t.numel() != n or t.dim() != 1 or t.get_device() != device or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous {dtype} tensor [{n}] on cuda:{device}, got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device}")


def _chk_device(t, name: str) -> int:
    """The index of a CUDA tensor's device, which has to be the current one (the call runs on its stream)."""
    i = t.get_device()
    if i < 0 or i != _current_device():
        raise RuntimeError(f"{name} must be on the current CUDA device, got {t.device}")
    return i


def _chk_table(t, device: int):
    """Block table int32 [B, pages] with contiguous rows that do not overlap -> (B, pages, row stride)."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.get_device() != device:
        raise RuntimeError("block_table must be an int32 CUDA tensor [B, pages] with contiguous rows")
    (B, width), (ld, step) = t.shape, t.stride()
    if width > 1 and step != 1:
        raise RuntimeError("block_table must be an int32 CUDA tensor [B, pages] with contiguous rows")
    if B <= 1:
        ld = width
    elif ld < width:
        raise RuntimeError("block_table rows must not overlap")
    return B, width, ld


def paged_plan_cuda(context_lens, new_lens, block_table, free_pages, free_head, page_size: int, max_tokens: int,
                    parents=None, max_new: Optional[int] = None) -> PagedPlan:
    """Plan of one decoding step for B requests with ``context_lens`` cached
    and ``new_lens`` new tokens (int32 [B]), built on the device.

    The pages that the new tokens need are taken in request order from
    ``free_pages`` (int32) starting at ``free_head`` (int32 [1]) and written
    into ``block_table`` (int32 [B, pages], updated in place) behind the pages
    that the context occupies. With ``parents`` (int32 [max_tokens]: for each
    row the index, within its request, of the token it follows, -1 for the
    context) the new tokens form trees of at most ``max_new`` tokens, and the
    plan holds their ancestor masks. Nothing is read on the host: what does
    not fit is reported in ``status``."""
    dev = _chk_device(context_lens, "context_lens")
    B, width, ld = _chk_table(block_table, dev)
    _chk1(context_lens, "context_lens", torch.int32, B, dev)
    _chk1(new_lens, "new_lens", torch.int32, B, dev)
    n_free = free_pages.numel()
    _chk1(free_pages, "free_pages", torch.int32, n_free, dev)
    _chk1(free_head, "free_head", torch.int32, 1, dev)
    if max_tokens < 0:
        raise RuntimeError("max_tokens must not be negative")
    words = 0
    if parents is not None:
        _chk1(parents, "parents", torch.int32, max_tokens, dev)
        if max_new is None or max_new < 1:
            raise RuntimeError("parents need max_new, the most new tokens of a request")
        words = (max_new + 31) // 32
    # one allocation for the small outputs: a view is cheaper than an allocation
    slots = new_lens.new_empty(max_tokens, dtype=torch.int64)
    mask = new_lens.new_empty((max_tokens, words)) if words else None
    ints = new_lens.new_empty(max_tokens * 2 + B + 3)
    request, position, starts, head, status = ints.split_with_sizes((max_tokens, max_tokens, B + 1, 1, 1))
    p_req = ints.data_ptr()
    p_pos = p_req + 4 * max_tokens
    p_starts = p_pos + 4 * max_tokens
    p_head = p_starts + 4 * (B + 1)
    _call("iw_paged_plan", _PLAN_DESC, dev, context_lens.data_ptr(), new_lens.data_ptr(), B, block_table.data_ptr(), ld,
          width, free_pages.data_ptr(), n_free, free_head.data_ptr(), page_size, max_tokens,
          parents.data_ptr() if words else 0, max_new or 0, slots.data_ptr(), p_req, p_pos,
          mask.data_ptr() if words else 0, p_starts, p_head, p_head + 4)
    return PagedPlan(slots, request, position, starts, head, status, mask)


def _cache_checks(k_cache, v_cache, device: int):
    """Paged K/V caches int8 [pages, heads, page_size, D] of one layout (D
    contiguous, any order of the other axes)."""
    if k_cache.dtype != torch.int8 or v_cache.dtype != torch.int8:
        raise RuntimeError("k_cache and v_cache must be int8")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise RuntimeError("k_cache and v_cache must be [pages, heads, page_size, D]")
    if k_cache.get_device() != device or v_cache.get_device() != device:
        raise RuntimeError(f"k_cache and v_cache must be on cuda:{device}")
    st = k_cache.stride()
    if st != v_cache.stride() or st[3] != 1:
        raise RuntimeError("k_cache and v_cache must have equal strides and contiguous rows")
    return st


def paged_kv_write_cuda(k, v, slots, k_cache, v_cache) -> None:
    """Write new K/V rows (int8 [N, heads, D], head rows contiguous: columns
    of the fused projection's output may be passed as views) into the paged
    caches (int8 [pages, heads, page_size, D]) at ``slots`` (int64 [N],
    ``PagedPlan.slots``; rows with a negative slot are skipped), in place."""
    dev = _chk_device(k, "k")
    if k.dtype != torch.int8 or v.dtype != torch.int8 or k.dim() != 3 or k.shape != v.shape or v.get_device() != dev:
        raise RuntimeError("k and v must be int8 CUDA tensors [N, heads, D] of one shape")
    sk, sv = k.stride(), v.stride()
    if sk[2] != 1 or sv[2] != 1:
        raise RuntimeError("k and v must have contiguous head rows")
    N, H, D = k.shape
    st = _cache_checks(k_cache, v_cache, dev)
    P, Hc, page, Dc = k_cache.shape
    if Hc != H or Dc != D:
        raise RuntimeError(f"k_cache must have {H} heads of {D}, got {tuple(k_cache.shape)}")
    _chk1(slots, "slots", torch.int64, N, dev)
    _lib.call("iw_paged_kv_write", k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], slots.data_ptr(),
              k_cache.data_ptr(), v_cache.data_ptr(), st[0], st[1], st[2], P, page, N, H, D, _raw_stream(dev))


def tree_attention_cuda(q, k_cache, v_cache, block_table, context_lens, starts, qk_multiplier, qk_shift, frac_bits,
                        av_multiplier, av_shift, rsqrt_offset: int = 16, tree_mask=None, out=None):
    """The integer attention of ``attention_cuda`` for the new tokens of a
    ragged batch over the paged caches: q int8 [N, H, D] (D 64 or 128; rows
    ``starts[b]:starts[b+1]`` belong to request b) -> int8 [N, H*D].

    The new tokens' own K/V are in the caches already
    (``paged_kv_write_cuda``). Each row sees its request's whole context and,
    of the new tokens, those whose bit ``tree_mask`` (int32 [N, words]) sets;
    without a mask itself and those before it. The caches may have fewer
    heads than q (query head h reads head h // (H / heads)). Rows from
    ``starts[B]`` on are padding and give 0."""
    dev = _chk_device(q, "q")
    if q.dtype != torch.int8 or q.dim() != 3 or q.stride(2) != 1:
        raise RuntimeError("q must be an int8 CUDA tensor [N, H, D] with contiguous head rows")
    N, H, D = q.shape
    st = _cache_checks(k_cache, v_cache, dev)
    P, Hkv, page, Dk = k_cache.shape
    if Dk != D:
        raise RuntimeError(f"head dimension mismatch: q has {D}, the caches {Dk}")
    if Hkv < 1 or H % Hkv:
        raise RuntimeError(f"the caches' head count {Hkv} must divide the query head count {H}")
    B, width, ld = _chk_table(block_table, dev)
    _chk1(context_lens, "context_lens", torch.int32, B, dev)
    _chk1(starts, "starts", torch.int32, B + 1, dev)
    p_mask = words = 0
    if tree_mask is not None:
        if (tree_mask.dtype != torch.int32 or tree_mask.dim() != 2 or tree_mask.shape[0] != N or tree_mask.shape[1] < 1
                or tree_mask.get_device() != dev or not tree_mask.is_contiguous()):
            raise RuntimeError("tree_mask must be a contiguous int32 CUDA tensor [N, words]")
        p_mask, words = tree_mask.data_ptr(), tree_mask.shape[1]
    if out is None:
        out = q.new_empty((N, H * D))
    elif out.dtype != torch.int8 or out.shape != (N, H * D) or out.get_device() != dev or out.stride(1) != 1:
        raise RuntimeError(f"out must be an int8 CUDA tensor [{N}, {H * D}] with contiguous rows")
    _call("iw_tree_attention", _ATTN_DESC, dev, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0),
          k_cache.data_ptr(), v_cache.data_ptr(), st[0], st[1], st[2], P, page, block_table.data_ptr(), ld, width,
          context_lens.data_ptr(), starts.data_ptr(), p_mask, words, B, N, H, Hkv, D,
          _scalar(qk_multiplier, "qk_multiplier"), _scalar(qk_shift, "qk_shift"), _scalar(frac_bits, "frac_bits"),
          _scalar(av_multiplier, "av_multiplier"), _scalar(av_shift, "av_shift"), rsqrt_offset)
    return out


_LOGITS = {torch.int8: 0, torch.float16: 1, torch.bfloat16: 2, torch.float32: 3}


class _Ungraded(torch.autograd.Function):
    """The scores of logits that ask for a gradient: asking them for it is an error."""

    @staticmethod
    def forward(ctx, logits, *args):
        return token_logprobs_cuda(logits, *args)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("token_logprobs_cuda has no gradient: it is for inference")


def token_logprobs_cuda(logits, targets=None, top: int = 0, scale: float = 1.0, suppress_bits=None):
    """Log probabilities of given tokens under softmax(scale * logits).

    logits [N, V] int8 (the classifier's; scale = 1/alpha), float16, bfloat16
    or float32 with contiguous rows; targets int64 [N, C] (negative: padding,
    gives 0; V or more: NaN); ``top`` alternatives per row (at most 32);
    suppress_bits int32 or uint32 [ceil(V/32)] removes token ids from every row.
    Returns (logprobs float32 [N, C], entropy float32 [N], top_ids int64
    [N, top], top_logprobs float32 [N, top]); equal logits are ordered by id,
    and an alternative that does not exist (fewer tokens than ``top`` with a
    logit above -inf) has id -1 and -inf. A row with a NaN or +inf gives NaN.
    For inference: there is no gradient, and a backward pass through the
    scores of logits that ask for one raises."""
    if logits.requires_grad and torch.is_grad_enabled():
        return _Ungraded.apply(logits, targets, top, scale, suppress_bits)
    dev = _chk_device(logits, "logits")
    if logits.dtype not in _LOGITS:
        raise RuntimeError(f"logits must be int8, float16, bfloat16 or float32, got {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise RuntimeError("logits must be [N, V] with contiguous rows")
    N, V = logits.shape
    n_given = p_targets = p_suppress = 0
    if targets is not None:
        if (targets.dtype != torch.int64 or targets.dim() != 2 or targets.shape[0] != N or targets.get_device() != dev
                or not targets.is_contiguous()):
            raise RuntimeError("targets must be a contiguous int64 CUDA tensor [N, C]")
        n_given = targets.shape[1]
        p_targets = targets.data_ptr() if n_given else 0
    if suppress_bits is not None:
        if suppress_bits.dtype not in (torch.int32, torch.uint32):
            raise RuntimeError(f"suppress_bits must be int32 or uint32, got {suppress_bits.dtype}")
        _chk1(suppress_bits, "suppress_bits", suppress_bits.dtype, (V + 31) // 32, dev)
        p_suppress = suppress_bits.data_ptr()
    if top < 0 or top > min(V, _lib.LOGPROBS_MAX_TOP):
        raise RuntimeError(f"top must be in [0, min(V, {_lib.LOGPROBS_MAX_TOP})], got {top}")
    lp = logits.new_empty((N, n_given), dtype=torch.float32)
    entropy = lp.new_empty(N)
    ids = logits.new_empty((N, top), dtype=torch.int64)
    top_lp = lp.new_empty((N, top))
    _call("iw_token_logprobs", _LOGP_DESC, dev, logits.data_ptr(), logits.stride(0) if N > 1 else V,
          _LOGITS[logits.dtype], N, V, scale, p_suppress, p_targets, n_given, top, lp.data_ptr(), entropy.data_ptr(),
          ids.data_ptr(), top_lp.data_ptr())
    return lp, entropy, ids, top_lp
