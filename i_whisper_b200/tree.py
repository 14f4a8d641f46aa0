"""Decoding with drafted token trees over a paged INT8 cache.

``TreeDecoder`` runs the decoder of a ``WhisperIntB200`` on ragged batches:
in one pass each utterance gets its own number of new tokens, which form a
chain (a prompt, one next token) or a tree of drafts hanging from its last
token. A pass is

  plan (pages, slots, positions, ancestor masks)      ops.paged_plan_cuda
  per layer: LN, QKV product, cache write,            ops.paged_kv_write_cuda
             self attention over the pages,           ops.tree_attention_cuda
             cross attention, MLP
  classifier, scores of every node                    ops.token_logprobs_cuda

with the products and LayerNorms of the model runner. The arithmetic is the
model's integer arithmetic, so every node's logits are the bytes that decoding
its path token by token gives, and a greedy walk through drafts gives the
tokens that greedy decoding gives. The reference's timestamp filters
are not applied: scores are over the raw logits (less ``suppress`` ids).

Cross attention uses the same operator on the cross K/V as the projection
writes them (head-major [H, B, n_audio_ctx, 64]), seen as pages without a copy.
"""
from __future__ import annotations

from typing import Callable, List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib, ops
from .model import WhisperIntB200, _rs


class TreeScores(NamedTuple):
    """What a pass says about its nodes, row by row in request order."""
    logits: torch.Tensor        # [N, n_vocab] int8 (a view of rows of n_vocab_pad)
    logprobs: torch.Tensor      # [N, C] float32 of the given targets
    entropy: torch.Tensor       # [N] float32
    top_ids: torch.Tensor       # [N, top] int64
    top_logprobs: torch.Tensor  # [N, top] float32
    plan: ops.PagedPlan


class TreeDecoder:
    """Paged decoding state of a batch of utterances.

    ``xa`` [B, n_audio_ctx, d] int8: the encoder's features (``model.encoder``; any
    strides, so that ``xa[:1].expand(8, -1, -1)`` decodes one utterance eight times;
    ``rs_xa``: their row sums, needed only where the checkpoint's zero points
    are not folded). ``pages`` pages of ``page_size`` tokens are shared by
    the batch (default: enough for every utterance's whole text context)."""

    def __init__(self, model: WhisperIntB200, xa: torch.Tensor, rs_xa: Optional[torch.Tensor] = None,
                 page_size: int = 16, pages: Optional[int] = None):
        dm = model.dims
        if xa.dtype != torch.int8 or xa.dim() != 3 or xa.shape[1:] != (dm.n_audio_ctx, dm.n_audio_state):
            raise RuntimeError("xa must be int8 features [B, n_audio_ctx, n_audio_state]")
        self.model, self.page_size = model, page_size
        self.B = B = xa.shape[0]
        dev = xa.device
        H, L, Ta = dm.n_text_head, dm.n_text_layer, dm.n_audio_ctx
        width = -(-dm.n_text_ctx // page_size)
        pages = B * width if pages is None else pages
        i32 = lambda n, v=0: torch.full((n,), v, dtype=torch.int32, device=dev)
        self.cache = torch.empty(L, 2, pages, H, page_size, 64, dtype=torch.int8, device=dev)
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.head = i32(1)
        self.ctx = i32(B)
        self.lens = [0] * B  # the context lengths on the host
        # cross K/V: rows of an utterance follow one another, so any power of two
        # that divides n_audio_ctx cuts them into pages
        page = Ta & -Ta
        ws = dict(cross=torch.empty(L * 2 * H * B * Ta * 64, dtype=torch.int8, device=dev))
        model.cross_kv(xa.contiguous(), rs_xa, ws)  # which takes its rows one after another
        self.cross = ws["cross"].view(L, 2, H, B * Ta // page, page, 64).permute(0, 1, 3, 2, 4, 5)
        self.cross_table = torch.arange(B * Ta // page, dtype=torch.int32, device=dev).view(B, Ta // page)
        self.cross_ctx = i32(B, Ta)
        self.suppress = model.suppress_bits
        self._plan = None

    def step(self, tokens: Sequence[Sequence[int]], parents: Optional[Sequence[Sequence[int]]] = None, top: int = 1,
             targets: Optional[torch.Tensor] = None, suppress: bool = False) -> TreeScores:
        """One pass over ``tokens[b]``, the new tokens of utterance b (none is
        allowed). With ``parents``, ``parents[b][i]`` is the index in
        ``tokens[b]`` of the token that token i follows, -1 for the context;
        without, each list is a chain. The context is not advanced
        (``accept`` does that)."""
        m, dm = self.model, self.model.dims
        if len(tokens) != self.B:
            raise RuntimeError(f"tokens must have {self.B} lists")
        n_new = [len(t) for t in tokens]
        N, most = sum(n_new), max(n_new)
        if N == 0:
            raise RuntimeError("no tokens")
        ids = [t for row in tokens for t in row]
        if min(ids) < 0 or max(ids) >= dm.n_vocab:
            raise RuntimeError(f"token ids must be in [0, {dm.n_vocab})")
        if any(c + n > dm.n_text_ctx for c, n in zip(self.lens, n_new)):
            raise RuntimeError(f"more than {dm.n_text_ctx} text tokens")
        dev = self.ctx.device
        flat = torch.tensor(ids, dtype=torch.int64).to(dev, non_blocking=True)
        up = None
        if parents is not None:
            if [len(p) for p in parents] != n_new:
                raise RuntimeError("parents must have the lists of tokens")
            up = torch.tensor([p for row in parents for p in row], dtype=torch.int32).to(dev, non_blocking=True)
        new = torch.tensor(n_new, dtype=torch.int32).to(dev, non_blocking=True)
        self._plan = None  # nothing to accept until this pass is through
        plan = ops.paged_plan_cuda(self.ctx, new, self.table, self.free, self.head, self.page_size, N, parents=up,
                                   max_new=most if up is not None else None)
        # pages run out only when the caller gave fewer than the batch can need
        if self.free.numel() < self.B * self.table.shape[1] and plan.status.item() & _lib.PLAN_POOL_EXHAUSTED:
            raise RuntimeError("out of cache pages")

        d, H = dm.n_text_state, dm.n_text_head
        e8 = lambda *s: torch.empty(*s, dtype=torch.int8, device=dev)
        rs = torch.empty(N, dtype=torch.int32, device=dev)
        h, qkv, q, att, f1 = e8(N, d), e8(N, 3 * d), e8(N, d), e8(N, d), e8(N, 4 * d)
        no_new = torch.zeros(N, 1, dtype=torch.int32, device=dev)  # cross attention sees no new tokens
        st = torch.cuda.current_stream().cuda_stream

        def att_sums(lin):
            if lin.wz is not None:
                _lib.call("iw_rowsum_i8", att.data_ptr(), d, N, d, rs.data_ptr(), st)
            return rs

        x16 = ops.add_requant15_cuda(m.tok_emb[flat][None], m.dec_pe[plan.position.long()], m.dec_m, m.dec_s)[0]
        i8, res = _lib.IW_GEMM_INT8, _lib.IW_GEMM_LINEAR32_RES
        for l, L in enumerate(m.dec_layers):
            m._ln(L["attn_ln"], x16, N, h, rowsum_out=_rs(L["qkv"], rs))
            m._gemm(h, d, N, L["qkv"], qkv, 3 * d, i8, rowsum=rs)
            qv, kv, vv = (qkv[:, i * d:(i + 1) * d].view(N, H, 64) for i in range(3))
            ops.paged_kv_write_cuda(kv, vv, plan.slots, self.cache[l, 0], self.cache[l, 1])
            a = L["attn"]
            ops.tree_attention_cuda(qv, self.cache[l, 0], self.cache[l, 1], self.table, self.ctx, plan.starts, a.qk_m, a.qk_s,
                                    a.fb, a.av_m, a.av_s, rsqrt_offset=m.RSQRT_OFFSET, tree_mask=plan.tree_mask, out=att)
            m._gemm(att, d, N, L["out"], x16, d, res, rowsum=att_sums(L["out"]), residual=x16, res_mult=L["attn_res"])
            m._ln(L["cross_ln"], x16, N, h, rowsum_out=_rs(L["cq"], rs))
            m._gemm(h, d, N, L["cq"], q, d, i8, rowsum=rs)
            a = L["cattn"]
            ops.tree_attention_cuda(q.view(N, H, 64), self.cross[l, 0], self.cross[l, 1], self.cross_table, self.cross_ctx,
                                    plan.starts, a.qk_m, a.qk_s, a.fb, a.av_m, a.av_s, rsqrt_offset=m.RSQRT_OFFSET,
                                    tree_mask=no_new, out=att)
            m._gemm(att, d, N, L["cout"], x16, d, res, rowsum=att_sums(L["cout"]), residual=x16, res_mult=L["cross_res"])
            m._ln(L["mlp_ln"], x16, N, h, rowsum_out=_rs(L["fc1"], rs))
            rs_f1 = torch.zeros(N, dtype=torch.int32, device=dev) if L["fc2"].wz is not None else None
            m._gemm(h, d, N, L["fc1"], f1, 4 * d, i8, rowsum=rs, gelu_tab=L["gelu_tab"], out_rowsum=rs_f1)
            m._gemm(f1, 4 * d, N, L["fc2"], x16, d, res, rowsum=rs_f1, residual=x16, res_mult=L["mlp_res"])
        m._ln(m.dec_ln, x16, N, h)
        logits = e8(N, m.n_vocab_pad)
        m._gemm(h, d, N, m.clf, logits, m.n_vocab_pad, i8)
        logits = logits[:, :dm.n_vocab]
        scores = ops.token_logprobs_cuda(logits, targets, top=top, scale=1.0 / m.logit_alpha,
                                         suppress_bits=self.suppress if suppress else None)
        self._granted = [-(-(c + n) // self.page_size) for c, n in zip(self.lens, n_new)]
        self._plan, self._n_new = plan, n_new
        # what each token follows, by the plan's rule: no earlier token counts as the context
        self._up = [[p if 0 <= p < i else -1 for i, p in enumerate(row)]
                    for row in ([range(-1, n - 1) for n in n_new] if parents is None else parents)]
        return TreeScores(logits, *scores, plan)

    def accept(self, paths: Sequence[Sequence[int]]) -> None:
        """Advance each utterance's context by the nodes ``paths[b]`` of the
        last pass (indices into its tokens, the first a child of the context,
        each the parent of the next: other nodes' K/V rows were computed under
        another history): their K/V rows are moved together behind the context,
        and pages that the rest had taken go back to the pool."""
        if self._plan is None:
            raise RuntimeError("no pass to accept paths of")
        if len(paths) != self.B:
            raise RuntimeError(f"accept needs {self.B} paths, an empty one where nothing is kept")
        plan, n_new, dev, page = self._plan, self._n_new, self.ctx.device, self.page_size
        src, dst, back = [], [], []
        start = 0
        for b, path in enumerate(paths):
            if any(not 0 <= i < n_new[b] for i in path) or any(i >= j for i, j in zip(path, path[1:])):
                raise RuntimeError("a path must be increasing indices of the utterance's new tokens")
            if [self._up[b][i] for i in path] != [-1, *path][:len(path)]:
                raise RuntimeError("a path must be a branch of the utterance's tree from the context downwards")
            for k, i in enumerate(path):
                if i != k:
                    src.append(start + i)
                    dst.append(start + k)
            start += n_new[b]
            kept = -(-(self.lens[b] + len(path)) // page)
            back += [b * self.table.shape[1] + c for c in range(kept, self._granted[b])]
        if src:
            s = plan.slots[torch.tensor(src, device=dev)]
            d = plan.slots[torch.tensor(dst, device=dev)]
            for layer in self.cache:
                rows = [x[s // page, :, s % page] for x in layer]  # gathered before anything is overwritten
                ops.paged_kv_write_cuda(rows[0], rows[1], d, layer[0], layer[1])
        self.head = plan.free_head
        if back:
            idx = torch.tensor(back, device=dev)
            at = self.head - len(back)
            self.free[(at + torch.arange(len(back), device=dev)).long()] = self.table.view(-1)[idx]
            self.table.view(-1)[idx] = -1
            self.head = at.to(torch.int32)
        self.lens = [c + len(p) for c, p in zip(self.lens, paths)]
        self.ctx = torch.tensor(self.lens, dtype=torch.int32).to(dev, non_blocking=True)
        self._plan = None

    def greedy(self, prompts: Sequence[Sequence[int]], n_tokens: int,
               draft: Callable[[int, List[int]], Tuple[List[int], List[int]]], suppress: bool = True) -> List[List[int]]:
        """Greedy decoding of ``n_tokens`` tokens per utterance, checked in
        drafted trees: ``draft(b, history)`` returns the drafted tokens and
        parents (-1: follows the history) that may continue utterance b. Returns
        the new tokens (fewer where the text context is full), the same
        whatever is drafted; good drafts take fewer passes (``self.passes``)."""
        hist = [list(p) for p in prompts]
        if not all(hist):
            raise RuntimeError("greedy needs a prompt of at least one token for every utterance")
        out: List[List[int]] = [[] for _ in prompts]
        self.passes = 0
        first = self.step(hist, suppress=suppress)
        self.accept([range(len(p)) for p in hist])
        ends = np.cumsum([len(p) for p in hist]) - 1
        best = first.top_ids[torch.from_numpy(ends).to(self.ctx.device), 0].tolist()
        for b, t in enumerate(best):
            out[b].append(t)
            hist[b].append(t)
        while any(len(o) < n_tokens for o in out):
            # each tree: the last token, not in the cache yet, and the drafts below it
            tokens, parents = [], []
            for b in range(self.B):
                left = min(n_tokens - len(out[b]), self.model.dims.n_text_ctx - self.lens[b])
                if left <= 0:
                    tokens.append([]), parents.append([])
                    continue
                t, p = draft(b, list(hist[b]))
                room = self.model.dims.n_text_ctx - self.lens[b] - 1
                t, p = t[:room], p[:room]
                tokens.append([hist[b][-1]] + list(t))
                parents.append([-1] + [i + 1 for i in p])
            if not any(tokens):
                break
            best = self.step(tokens, parents, suppress=suppress).top_ids[:, 0].tolist()
            self.passes += 1
            paths, start = [], 0
            for b in range(self.B):
                path = [0] if tokens[b] else []
                while path and len(out[b]) < n_tokens:
                    nxt = best[start + path[-1]]
                    out[b].append(nxt)
                    hist[b].append(nxt)
                    child = [i for i in range(path[-1] + 1, len(tokens[b]))
                             if parents[b][i] == path[-1] and tokens[b][i] == nxt]
                    if not child:
                        break
                    path.append(child[0])
                # the last token found is not in the cache: it roots the next tree
                paths.append(path)
                start += len(tokens[b])
            self.accept(paths)
        return [o[:n_tokens] for o in out]


def main() -> None:
    """Greedy decoding of a few synthetic windows with and without drafts (the
    drafts: the plain run's own continuation among wrong tokens, as a good draft
    model would give them)."""
    import time

    from .checkpoint import ModelDims, synthetic_state_dict
    from .synthetic import synthetic_mel_batch

    dims = ModelDims(80, 1500, 384, 6, 4, 51865, 448, 384, 6, 4)
    sd = synthetic_state_dict(dims, seed=0)
    mel = torch.from_numpy(synthetic_mel_batch(dims.n_mels, range(8), float(sd["encoder.input_alpha"][0]))).cuda()
    model = WhisperIntB200(dims, sd)
    xa = model.encoder(mel)
    prompts, n = [list(model.tokens_spec["sot_sequence"])] * 8, 64
    rng = np.random.default_rng(0)
    plain: List[List[int]] = []

    def nothing(b, hist):
        return [], []

    def good(b, hist):
        right = plain[b][len(hist) - len(prompts[b]):][:4]
        t, p, last = [], [], -1
        for tok in right:
            t += [int(rng.integers(0, dims.n_vocab)), tok]
            p += [last, last]
            last = len(t) - 1
        return t, p

    for name, draft in (("no drafts", nothing), ("trees of drafts", good)):
        TreeDecoder(model, xa).greedy(prompts, 8, draft)  # first run: kernel attributes
        dec = TreeDecoder(model, xa)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        out = dec.greedy(prompts, n, draft)
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        plain = plain or out
        print(f"{name}: {dec.passes + 1} passes, {8 * n / dt:.0f} tokens/s, "
              f"{'the same tokens' if out == plain else 'OTHER TOKENS'}")


if __name__ == "__main__":
    main()
