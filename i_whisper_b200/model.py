"""GPU-resident integer Whisper: encoder + greedy decoder on sm_100a.

``WhisperIntB200`` runs the forward of the reference ``Whisper_int``
(vcsd-lab/I-Whisper, i_whisper/model_int.py:1524-1618) with the dataflow of
AudioEncoder_int.forward (:1260-1316), ResidualAttentionBlock_int.forward
(:1112-1177), MultiHeadAttention_int (:677-1042) and TextDecoder_int.forward
(:1398-1484), bit for bit, but laid out for the GPU:

* each block is LN -> fused QKV GEMM -> attention -> out GEMM fused with
  Residual15 -> LN -> fc1 GEMM fused with GeLU -> fc2 GEMM fused with
  Residual15; the conv stem is two windowed GEMMs (the convolutions read
  their channels-last, zero-padded inputs in place, weights in (tap,
  channel) order) with GeLU and the positional add-requant fused into the
  epilogues;
* zero-point row sums come from the producer (LayerNorm, fc1 epilogue), so
  no GEMM re-reads its input for them;
* cross-attention K/V of every decoder layer are computed by one GEMM over
  the encoder output and stored head-major ``[L, 2, H, B, T, 64]``; the
  self-attention cache is preallocated ``[L, 2, B, H, n_text_ctx, 64]`` and
  appended in place (instead of the torch.cat of the reference's hooks);
* the greedy decode state lives on the device, so a decode step is a fixed
  kernel sequence that is captured once in a CUDA graph and replayed.

All kernels come from ``libiwhisper_b200.so`` through its C ABI.
"""
from __future__ import annotations

import ctypes as C
import json
import os
from dataclasses import dataclass
from typing import Dict, List, Optional

import numpy as np
import torch

from . import _lib
from .checkpoint import ModelDims, check_state_dict

_ASSETS = os.path.join(os.path.dirname(os.path.abspath(__file__)), "assets")


def decode_tokens(n_vocab: int) -> dict:
    """Special-token ids of the reference tokenizer for this vocabulary
    (generated by assets/make_decode_tokens.py)."""
    with open(os.path.join(_ASSETS, "decode_tokens.json")) as f:
        return json.load(f)[str(n_vocab)]


def _i(x) -> int:
    return int(np.asarray(x).reshape(-1)[0])


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    if t is None or isinstance(t, int):
        return t
    return t.data_ptr()


class KernelTimer:
    """Records a CUDA event pair on the launching stream around each launch
    of the runner (category, algorithmic work) for roofline accounting."""

    def __init__(self):
        self.records = []

    def start(self):
        ev = torch.cuda.Event(enable_timing=True)
        ev.record()
        return ev

    def stop(self, ev0, cat: str, ops: float = 0.0, nbytes: float = 0.0):
        ev1 = torch.cuda.Event(enable_timing=True)
        ev1.record()
        self.records.append((cat, ops, nbytes, ev0, ev1))

    def summary(self):
        torch.cuda.synchronize()
        out = {}
        for cat, ops, nb, a, b in self.records:
            r = out.setdefault(cat, {"launches": 0, "ms": 0.0, "ops": 0.0, "bytes": 0.0})
            r["launches"] += 1
            r["ms"] += a.elapsed_time(b)
            r["ops"] += ops
            r["bytes"] += nb
        return out


@dataclass
class _Linear:
    w: torch.Tensor
    bias: Optional[torch.Tensor]
    wz: Optional[torch.Tensor]
    mult: torch.Tensor
    shift: torch.Tensor
    sign: Optional[torch.Tensor] = None  # [N] int8 +1/-1 when the zero point is folded into w


def fold_zero_point(w: np.ndarray, wz: np.ndarray):
    """Fold a Linear_int weight zero point into the weights, exactly.

    Linear_int's accumulator is acc = sum_k x[k]*w[n,k] - wz[n]*sum_k x[k]
    (linear.py:50-97) = sum_k x[k]*(w[n,k] - wz[n]). With int8 w and wz the
    differences lie in [-255, 255]; where a channel's differences fit
    [-128, 127] they are the channel's new weights (sign +1), where their
    negations do, those are (sign -1: the GEMM multiplies that channel's
    accumulator by -1 before the bias). The GEMM then needs no row sums of
    its input. Returns (w' int8 [N, K], sign int8 [N]), or None when some
    channel fits neither way (the caller keeps the zero-point form)."""
    d = w.astype(np.int32).reshape(w.shape[0], -1) - np.asarray(wz, np.int32).reshape(-1, 1)
    fits = (d.min(1) >= -128) & (d.max(1) <= 127)
    fits_neg = (d.min(1) >= -127) & (d.max(1) <= 128)
    if not np.all(fits | fits_neg):
        return None
    sign = np.where(fits, 1, -1).astype(np.int8)
    return (d * sign.astype(np.int32)[:, None]).astype(np.int8).reshape(w.shape), sign


@dataclass
class _LN:
    gamma: torch.Tensor
    beta: Optional[torch.Tensor]
    ln_m: int
    ln_s: int
    out_m: int
    out_s: int


@dataclass
class _Gelu:
    lut: torch.Tensor
    mi: torch.Tensor
    si: torch.Tensor
    mo: torch.Tensor
    so: torch.Tensor


@dataclass
class _Attn:
    qk_m: int
    qk_s: int
    fb: int
    av_m: int
    av_s: int


def _rs(lin: "_Linear", buf: torch.Tensor) -> Optional[torch.Tensor]:
    """The row-sum buffer a producer fills for the GEMM `lin`, or None when
    that GEMM has no zero point to apply (folded into its weights)."""
    return buf if lin.wz is not None else None


class WhisperIntB200:
    """Integer Whisper forward on one GPU.

    ``state_dict`` is keyed exactly like ``Whisper_int.state_dict()`` (numpy
    arrays or CPU tensors), e.g. from ``checkpoint.load_int_checkpoint``.
    """

    RSQRT_OFFSET = 16  # MultiHeadAttention_int.rsqrt_offset (model_int.py:704)

    def __init__(self, dims: ModelDims, state_dict: Dict[str, object], device="cuda", layernorm: str = "32",
                 fold_zero_points: bool = True):
        sd = {k: (v.numpy() if isinstance(v, torch.Tensor) else np.asarray(v)) for k, v in state_dict.items()}
        check_state_dict(dims, sd)
        if layernorm not in ("32", "64"):
            raise ValueError("layernorm must be '32' (LayerNorm32) or '64' (the LayerNorm64 research variant)")
        # LayerNorm_int backend: "32" is the reference default; "64" its
        # scalar64/simd64 research variant (model_int.py:252-287)
        self._ln_entry = _lib.LIB.iw_layernorm32_ex if layernorm == "32" else _lib.LIB.iw_layernorm64_ex
        self.dims = dims
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("WhisperIntB200 runs on CUDA devices only")
        dev = self.device

        def T(a):
            return torch.from_numpy(np.ascontiguousarray(a)).to(dev)

        def make_lin(w, bias, wz, mult, shift) -> _Linear:
            # zero points folded into the weights where every channel allows
            # it (the reference-calibrated checkpoints: all layers)
            # (the row-major kernel, IW_GEMM_ROWMAJOR=1, has no accumulator signs)
            fold = fold_zero_points and wz is not None and os.environ.get("IW_GEMM_ROWMAJOR") != "1"
            folded = fold_zero_point(w, wz) if fold else None
            if folded is not None:
                return _Linear(T(folded[0]), bias, None, mult, shift, T(folded[1]))
            return _Linear(T(w), bias, T(wz) if wz is not None else None, mult, shift)

        def lin(pre, bias=True) -> _Linear:
            return make_lin(np.asarray(sd[pre + ".weight"]), T(sd[pre + ".bias"]) if pre + ".bias" in sd else None,
                            sd[pre + ".wgt_zeros"] if pre + ".wgt_zeros" in sd else None,
                            T(sd[pre + ".req_multiplier"]), T(sd[pre + ".req_shiftmount"]))

        def lin_cat(pres) -> _Linear:
            n = [sd[p + ".weight"].shape[0] for p in pres]
            bias = [sd[p + ".bias"] if p + ".bias" in sd else np.zeros(k, np.int32) for p, k in zip(pres, n)]
            return make_lin(np.concatenate([sd[p + ".weight"] for p in pres]), T(np.concatenate(bias)),
                            np.concatenate([sd[p + ".wgt_zeros"] for p in pres]),
                            T(np.concatenate([sd[p + ".req_multiplier"] for p in pres])),
                            T(np.concatenate([sd[p + ".req_shiftmount"] for p in pres])))

        def ln(pre) -> _LN:
            return _LN(T(sd[pre + ".weight"]), T(sd[pre + ".bias"]) if pre + ".bias" in sd else None,
                       _i(sd[pre + ".ln_req_multiplier"]), _i(sd[pre + ".ln_req_shiftmount"]),
                       _i(sd[pre + ".out_req_multiplier"]), _i(sd[pre + ".out_req_shiftmount"]))

        def gelu(pre) -> _Gelu:
            return _Gelu(T(sd[pre + ".lut"]), T(sd[pre + ".luti_req_multiplier"]), T(sd[pre + ".luti_req_shiftmount"]),
                         T(sd[pre + ".luto_req_multiplier"]), T(sd[pre + ".luto_req_shiftmount"]))

        def attn(pre) -> _Attn:
            return _Attn(_i(sd[pre + ".qk_req_multiplier"]), _i(sd[pre + ".qk_req_shiftmount"]),
                         _i(sd[pre + ".qk_frac_bits"]), _i(sd[pre + ".av_req_multiplier"]),
                         _i(sd[pre + ".av_req_shiftmount"]))

        # ---- encoder ----------------------------------------------------
        e = "encoder"
        def conv_taps_first(pre) -> _Linear:
            # Conv1d_int weight [cout, cin*3] (tap fastest, conv1d.h) reordered
            # to [cout, 3*cin] (channel fastest): the windowed GEMM reads the
            # three taps as three consecutive channels-last rows
            w = np.asarray(sd[pre + ".weight"])
            w = w.reshape(w.shape[0], -1, 3).transpose(0, 2, 1).reshape(w.shape[0], -1)
            return _Linear(T(np.ascontiguousarray(w)), T(sd[pre + ".bias"]) if pre + ".bias" in sd else None, None,
                           T(sd[pre + ".req_multiplier"]), T(sd[pre + ".req_shiftmount"]))

        self.conv1 = conv_taps_first(e + ".conv1")
        self.conv1_ms = (_i(sd[e + ".conv1.req_multiplier"]), _i(sd[e + ".conv1.req_shiftmount"]))
        self.conv2 = conv_taps_first(e + ".conv2")
        self.conv2_ms = (_i(sd[e + ".conv2.req_multiplier"]), _i(sd[e + ".conv2.req_shiftmount"]))
        self.gelu1, self.gelu2 = gelu(e + ".gelu1"), gelu(e + ".gelu2")
        self.enc_pe = T(sd[e + ".positional_embedding"])
        self.input_alpha = float(np.asarray(sd[e + ".input_alpha"], np.float32).reshape(-1)[0])
        self.enc_pm, self.enc_ps = T(sd[e + ".req_multiplier"]), T(sd[e + ".req_shiftmount"])
        self.enc_layers = []
        for i in range(dims.n_audio_layer):
            p = f"{e}.blocks.{i}"
            self.enc_layers.append(dict(
                attn_ln=ln(p + ".attn_ln"), qkv=lin_cat([p + ".attn.query", p + ".attn.key", p + ".attn.value"]),
                attn=attn(p + ".attn"), out=lin(p + ".attn.out"), attn_res=_i(sd[p + ".attn_res_req_multiplier"]),
                mlp_ln=ln(p + ".mlp_ln"), fc1=lin(p + ".mlp.0"), gelu=gelu(p + ".mlp.1"), fc2=lin(p + ".mlp.2"),
                mlp_res=_i(sd[p + ".mlp_res_req_multiplier"])))
        self.ln_post = ln(e + ".ln_post")
        # ---- decoder ----------------------------------------------------
        dd = "decoder"
        # The tied embedding doubles as the classifier weight. Its rows are
        # padded with zeros to a multiple of 32 so the classifier GEMM runs
        # the per-channel fast epilogue on 16-byte aligned logit rows; the
        # embedding gather never reads the padding, and the greedy step
        # scans only the first n_vocab logits of each row.
        V = dims.n_vocab
        self.n_vocab_pad = (V + 31) // 32 * 32
        emb = np.zeros((self.n_vocab_pad, dims.n_text_state), np.int8)
        emb[:V] = sd[dd + ".token_embedding.weight"]
        self.tok_emb = T(emb)
        self.dec_pe = T(sd[dd + ".positional_embedding"])
        self.dec_m = T(sd[dd + ".req_multiplier"].astype(np.uint16))
        self.dec_s = T(sd[dd + ".req_shiftmount"])
        cm, cs = _i(sd[dd + ".clf_req_multiplier"]), _i(sd[dd + ".clf_req_shiftmount"])
        # classifier_scalar shifts by max(shift, 0) (classifier_scalar.cpp:91-140)
        self.clf = _Linear(self.tok_emb, None, None, T(np.full(self.n_vocab_pad, cm, np.uint32)),
                           T(np.full(self.n_vocab_pad, max(cs, 0), np.int8)))
        self.logit_alpha = float(np.asarray(sd[dd + ".act_logits_alpha"], np.float32).reshape(-1)[0])
        self.dec_layers = []
        cross_pres = []
        for i in range(dims.n_text_layer):
            p = f"{dd}.blocks.{i}"
            cross_pres += [p + ".cross_attn.key", p + ".cross_attn.value"]
            self.dec_layers.append(dict(
                attn_ln=ln(p + ".attn_ln"), qkv=lin_cat([p + ".attn.query", p + ".attn.key", p + ".attn.value"]),
                attn=attn(p + ".attn"), out=lin(p + ".attn.out"), attn_res=_i(sd[p + ".attn_res_req_multiplier"]),
                cross_ln=ln(p + ".cross_attn_ln"), cq=lin(p + ".cross_attn.query"), cattn=attn(p + ".cross_attn"),
                cout=lin(p + ".cross_attn.out"), cross_res=_i(sd[p + ".cross_attn_res_req_multiplier"]),
                mlp_ln=ln(p + ".mlp_ln"), fc1=lin(p + ".mlp.0"), gelu=gelu(p + ".mlp.1"), fc2=lin(p + ".mlp.2"),
                mlp_res=_i(sd[p + ".mlp_res_req_multiplier"])))
        self.cross_kv_w = lin_cat(cross_pres)
        for L in self.enc_layers + self.dec_layers:
            # exact per-channel GeLU results for every int8 input (1 MiB per layer, twice)
            L["gelu_tab"] = self._gelu_table(L["gelu"], L["fc1"].w.shape[0])
        # shift-exp tables of the tensor-core attention, one per frac_bits
        # (every frac_bits fits: the whole table lives in shared memory)
        self._exp_tables = {}
        for L in self.enc_layers:
            fb = L["attn"].fb
            if fb not in self._exp_tables:
                tab = torch.empty(32772, dtype=torch.uint8, device=self.device)
                _lib.call("iw_shift_exp_table", fb, tab.data_ptr(), _stream())
                self._exp_tables[fb] = tab
        self.dec_ln = ln(dd + ".ln")
        tk = decode_tokens(dims.n_vocab)
        self.tokens_spec = tk
        bits = np.zeros((dims.n_vocab + 31) // 32, np.uint32)
        for t in tk["suppress"]:
            bits[t >> 5] |= np.uint32(1 << (t & 31))
        self.suppress_bits = T(bits)
        self.blank = T(np.array(tk["blank"], np.int32))
        self._enc_ws = {}
        self._dec_ws = {}
        self._graphs = {}
        self._enc_graphs = {}  # batch -> (CUDA graph, its input buffer, its output)
        self._pipe = {}  # batch -> (two input buffers, two output buffers, one CUDA graph per pair)
        self.graph_launches = {}  # (graph, batch) -> kernel launches captured in it
        self.replayed_launches = 0  # kernel launches run by replaying captured graphs
        self.timer: Optional[KernelTimer] = None  # set to a KernelTimer to time every launch
        self.launches = 0  # kernel launches issued by this runner (graph replays excluded)

    def _gelu_table(self, g: _Gelu, N: int) -> torch.Tensor:
        """(table [N, 256], the same rearranged for per-tile bulk copies)."""
        tab = torch.empty(N, 256, dtype=torch.int8, device=self.device)
        _lib.check(_lib.LIB.iw_gelu_table(g.lut.data_ptr(), g.mi.data_ptr(), g.si.data_ptr(), g.mo.data_ptr(),
                                          g.so.data_ptr(), g.mi.numel(), g.mo.numel(), N, tab.data_ptr(), _stream()))
        tiled = torch.empty((N + 127) // 128, 32768, dtype=torch.int8, device=self.device)
        _lib.check(_lib.LIB.iw_gelu_table_tiled(tab.data_ptr(), N, tiled.data_ptr(), _stream()))
        return tab, tiled

    # ------------------------------------------------------------------
    # kernel launch helpers
    # ------------------------------------------------------------------
    def _gemm(self, x, ldx, M, lin: _Linear, out, ldo, mode, rowsum=None, gelu: Optional[_Gelu] = None,
              gelu_pc=(1, 1), residual=None, res_mult=0, out_rowsum=None, headmajor=None, scalar=None, pos=None,
              gelu_tab=None, vt=None, kv=None, window=None):
        N, K = lin.w.shape
        d = _lib.GemmDesc()
        d.x, d.ldx, d.w, d.ldw, d.M, d.N, d.K = _ptr(x), ldx, lin.w.data_ptr(), K, M, N, K
        d.mode, d.out, d.ldo = mode, _ptr(out), ldo
        d.bias = _ptr(lin.bias)
        if lin.wz is not None and rowsum is not None:
            d.weight_zero, d.x_rowsum = lin.wz.data_ptr(), rowsum.data_ptr()
        elif lin.wz is not None:
            raise RuntimeError("zero-point row sums missing")
        if scalar is None:
            d.multiplier, d.shift = lin.mult.data_ptr(), lin.shift.data_ptr()
        else:
            d.scalar_multiplier, d.scalar_shift = scalar
        if gelu is not None:
            d.lut, d.luti_multiplier, d.luti_shift = gelu.lut.data_ptr(), gelu.mi.data_ptr(), gelu.si.data_ptr()
            d.luto_multiplier, d.luto_shift = gelu.mo.data_ptr(), gelu.so.data_ptr()
            d.luti_per_channel, d.luto_per_channel = gelu_pc
        if residual is not None:
            d.residual, d.ldr, d.residual_multiplier = residual.data_ptr(), ldo, res_mult
        if pos is not None:
            pe, pm, ps, T_ = pos
            d.pos, d.pos_T, d.pos_multiplier, d.pos_shift = pe.data_ptr(), T_, pm.data_ptr(), ps.data_ptr()
            d.pos_per_channel = 1 if pm.numel() > 1 else 0
        if headmajor is not None:
            d.headmajor_T, d.headmajor_B = headmajor
        d.out_rowsum = _ptr(out_rowsum)
        d.weight_sign = _ptr(lin.sign)
        if gelu_tab is not None:
            d.gelu_table, d.gelu_table_tiled = _ptr(gelu_tab[0]), _ptr(gelu_tab[1])
        if kv is not None:  # self-attention K/V straight into the caches
            d.kv_cache_k, d.kv_cache_v, d.kv_col0, d.kv_heads, d.kv_T, d.kv_Tcap, d.kv_pos, d.kv_pos_dev = kv
        if window is not None:  # (rows per window, bytes between windows): implicit convolution
            d.x_window_rows, d.x_window_stride = window
        if vt is not None:  # (V^T buffer, first V channel, rows per batch)
            vbuf, c0, T_ = vt
            d.vt_out, d.vt_ld, d.vt_col0, d.vt_T = vbuf.data_ptr(), vbuf.shape[1], c0, T_
        t = self.timer.start() if self.timer else None
        _lib.check(_lib.LIB.iw_gemm_i8(C.byref(d), _stream()))
        self.launches += 1
        if t is not None:
            self.timer.stop(t, "gemm_i8", ops=2.0 * M * N * K, nbytes=float(M * K + N * K))

    def _ln(self, p: _LN, x, rows, y, rowsum_out=None, rowsum_zero=None, ldx=None, ldy=None):
        d = p.gamma.numel()
        t = self.timer.start() if self.timer else None
        _lib.check(self._ln_entry(x.data_ptr(), ldx or d, p.gamma.data_ptr(), _ptr(p.beta), p.ln_m, p.ln_s,
                                              p.out_m, p.out_s, y.data_ptr(), ldy or d, rows, d, _ptr(rowsum_out),
                                              _ptr(rowsum_zero), _stream()))
        self.launches += 1
        if t is not None:
            self.timer.stop(t, "layernorm32", nbytes=3.0 * rows * d)

    def _attn(self, a: _Attn, B, H, Tq, Tk, q, q_str, k, k_str, v, v_str, y, y_str, mask_mode=0, Tk_dev=None,
              Tk_cap=0, vt=None, vt_ready=False, rowsum_out=None):
        d = _lib.AttnDesc()
        d.q, (d.ldq, d.q_bs, d.q_hs) = q, q_str
        d.k, (d.ldk, d.k_bs, d.k_hs) = k, k_str
        d.v, (d.ldv, d.v_bs, d.v_hs) = v, v_str
        d.y, (d.ldy, d.y_bs, d.y_hs) = y, y_str
        d.B, d.H, d.Tq, d.Tk = B, H, Tq, Tk
        d.Tk_dev, d.Tk_cap = _ptr(Tk_dev), Tk_cap
        d.mask_mode = mask_mode
        d.row_sum_out = _ptr(rowsum_out)
        d.qk_multiplier, d.qk_shift, d.frac_bits = a.qk_m, a.qk_s, a.fb
        d.av_multiplier, d.av_shift, d.rsqrt_offset = a.av_m, a.av_s, self.RSQRT_OFFSET
        if vt is not None and a.fb in self._exp_tables:
            d.exp_table, d.vt, d.vt_ld = self._exp_tables[a.fb].data_ptr(), vt.data_ptr(), vt.shape[1]
            d.vt_ready = 1 if vt_ready else 0
        t = self.timer.start() if self.timer else None
        _lib.check(_lib.LIB.iw_attention_ex(C.byref(d), _stream()))
        self.launches += 1
        if t is not None:
            # QK^T and P.V counted once each: 2 * 2 * B*H*Tq*Tk*64
            self.timer.stop(t, "attention", ops=4.0 * B * H * Tq * Tk * 64, nbytes=float(B * H * (Tq + 2 * Tk) * 64))

    # ------------------------------------------------------------------
    # encoder
    # ------------------------------------------------------------------
    def _enc_workspace(self, B):
        if B in self._enc_ws:
            return self._enc_ws[B]
        dm, dev = self.dims, self.device
        d, T = dm.n_audio_state, dm.n_audio_ctx
        Tm = 2 * T
        e8 = lambda *s: torch.empty(*s, dtype=torch.int8, device=dev)
        e32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)
        H = dm.n_audio_head
        # conv stem operands: the mel channels-last with 2 zero rows before
        # and 1 after each window; conv1's output with one extra row (t = -1,
        # zeroed) before each window
        ws = dict(mel_cl=e8(B * (Tm + 3), dm.n_mels), x1p=e8(B * (Tm + 1), d),
                  x16=torch.empty(B * T, d, dtype=torch.int16, device=dev), h=e8(B * T, d), rs_h=e32(B * T),
                  qkv=e8(B * T, 3 * d), att=e8(B * T, d), rs_att=e32(B * T), f1=e8(B * T, 4 * d), rs_f1=e32(B * T),
                  xa=e8(B, T, d), rs_xa=e32(B * T), vt=e8(B * H * 64, (T + 15) // 16 * 16))
        self._enc_ws[B] = ws
        return ws

    def encoder_graphed(self, mel_i8: torch.Tensor) -> torch.Tensor:
        """``encoder`` replayed from a CUDA graph captured once per batch
        size: the mel is copied into a fixed input buffer, every kernel of the
        encoder is one graph launch, and the result aliases the internal
        output buffer (as ``encoder`` without ``out``). Small batches, whose
        encoder time is otherwise the host's launch time, gain most; the
        bytes are the same as ``encoder``'s."""
        if mel_i8.dtype != torch.int8 or not mel_i8.is_cuda or not mel_i8.is_contiguous() or mel_i8.dim() != 3:
            raise RuntimeError("mel must be a contiguous int8 CUDA tensor [B, n_mels, frames]")
        B = mel_i8.shape[0]
        entry = self._enc_graphs.get(B)
        if entry is None:
            static_in = torch.empty_like(mel_i8)
            static_in.copy_(mel_i8)
            self.encoder(static_in)  # first run: workspaces and kernel attributes outside the capture
            st = torch.cuda.Stream()
            st.wait_stream(torch.cuda.current_stream())
            g = torch.cuda.CUDAGraph()
            timer, self.timer = self.timer, None  # no per-launch events inside the graph
            n0 = self.launches
            try:
                with torch.cuda.stream(st):
                    with torch.cuda.graph(g, stream=st):
                        xa = self.encoder(static_in)
            finally:
                self.timer = timer
            self.graph_launches[("encoder", B)] = self.launches - n0
            self.launches = n0
            torch.cuda.current_stream().wait_stream(st)
            entry = self._enc_graphs[B] = (g, static_in, xa)
        g, static_in, xa = entry
        if mel_i8.data_ptr() != static_in.data_ptr():
            static_in.copy_(mel_i8)
        g.replay()
        self.replayed_launches += self.graph_launches[("encoder", B)]
        return xa

    def encoder(self, mel_i8: torch.Tensor, trace: Optional[dict] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """AudioEncoder_int.forward on an INT8 mel [B, n_mels, 2*n_audio_ctx]
        (CUDA) -> INT8 features [B, n_audio_ctx, d]. Without ``out`` the result
        aliases an internal buffer that the next call for the same batch
        overwrites; with ``out`` (contiguous int8 CUDA [B, n_audio_ctx, d]) it is
        written there."""
        dm = self.dims
        if mel_i8.dtype != torch.int8 or not mel_i8.is_cuda or not mel_i8.is_contiguous():
            raise RuntimeError("mel must be a contiguous int8 CUDA tensor")
        B, n_mels, Tm = mel_i8.shape
        T, d, H = dm.n_audio_ctx, dm.n_audio_state, dm.n_audio_head
        if n_mels != dm.n_mels or Tm != 2 * T:
            raise RuntimeError("incorrect audio shape")
        ws = self._enc_workspace(B)
        st = _stream()
        M = B * T
        # conv1 (k=3, pad 1, stride 1) + GeLU1 as a windowed GEMM: output row
        # t' of a window (t = t' - 1, t' in [0, Tm]) reads the channels-last
        # mel rows t'..t'+2 (x[t-1..t+1]) as one 3*n_mels-wide row
        _lib.check(_lib.LIB.iw_channels_last_pad(mel_i8.data_ptr(), B, n_mels, Tm, 2, 1, ws["mel_cl"].data_ptr(),
                                                 st))
        self.launches += 1
        self._gemm(ws["mel_cl"], n_mels, B * (Tm + 1), self.conv1, ws["x1p"], d, _lib.IW_GEMM_INT8,
                   scalar=self.conv1_ms, gelu=self.gelu1, gelu_pc=(0, 0), window=(Tm + 1, (Tm + 3) * n_mels))
        # row t' = 0 (t = -1) becomes conv2's zero padding
        _lib.check(_lib.LIB.iw_zero_rows(ws["x1p"].data_ptr(), B, d, (Tm + 1) * d, st))
        self.launches += 1
        # conv2 (stride 2) + GeLU2 + positional add-requant -> INT15 residual:
        # output row t reads conv1 rows 2t-1..2t+1 (rows 2t..2t+2 of x1p)
        self._gemm(ws["x1p"], 2 * d, M, self.conv2, ws["x16"], d, _lib.IW_GEMM_INT8, scalar=self.conv2_ms,
                   gelu=self.gelu2, gelu_pc=(0, 1), pos=(self.enc_pe, self.enc_pm, self.enc_ps, T),
                   window=(T, (Tm + 1) * d))
        if trace is not None:
            trace["encoder.pos"] = ws["x16"].clone()
        for i, L in enumerate(self.enc_layers):
            self._block(L, ws, B, T, H, d)
            if trace is not None:
                trace[f"encoder.blocks.{i}"] = ws["x16"].clone()
        if out is not None:
            if out.dtype != torch.int8 or not out.is_cuda or not out.is_contiguous() or out.numel() != M * d:
                raise RuntimeError("out must be a contiguous int8 CUDA tensor [B, n_audio_ctx, d]")
        xa = ws["xa"] if out is None else out
        self._ln(self.ln_post, ws["x16"], M, xa, rowsum_out=_rs(self.cross_kv_w, ws["rs_xa"]))
        return xa

    def encoder_from_audio(self, audio: torch.Tensor) -> torch.Tensor:
        """The encoder on float32 16 kHz CUDA audio [B, 480000]: the GPU
        log-mel frontend (frontend.log_mel_int8_cuda, the reference's
        log_mel_spectrogram + input quantisation) then ``encoder``."""
        from .frontend import log_mel_int8_cuda
        return self.encoder(log_mel_int8_cuda(audio, self.dims.n_mels, self.input_alpha))

    def _pipe_slots(self, mel_shape, feat_shape):
        """Two device input/output buffer pairs for ``encode_batches`` at one
        batch size, with one CUDA graph per pair (the encoder reading input
        s and writing output s), captured once and kept."""
        B = mel_shape[0]
        ent = self._pipe.get(B)
        if ent is None:
            dev = self.device
            d_in = [torch.zeros(mel_shape, dtype=torch.int8, device=dev) for _ in range(2)]
            d_out = [torch.empty(feat_shape, dtype=torch.int8, device=dev) for _ in range(2)]
            self.encoder(d_in[0], out=d_out[0])  # first run: workspaces and kernel attributes outside the capture
            st = torch.cuda.Stream(dev)
            st.wait_stream(torch.cuda.current_stream(dev))
            graphs = []
            timer, self.timer = self.timer, None  # no per-launch events inside the graphs
            n0 = self.launches
            try:
                for k in range(2):
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.stream(st):
                        with torch.cuda.graph(g, stream=st):
                            self.encoder(d_in[k], out=d_out[k])
                    graphs.append(g)
            finally:
                self.timer = timer
            self.graph_launches[("encode_batches", B)] = (self.launches - n0) // 2
            self.launches = n0
            torch.cuda.current_stream(dev).wait_stream(st)
            ent = self._pipe[B] = (d_in, d_out, graphs)
        return ent

    def encode_batches(self, host_mels: List[torch.Tensor], host_feats: List[torch.Tensor]) -> None:
        """Encoder over a sequence of batches held in (pinned) host memory:
        host_feats[i] receives the INT8 features of host_mels[i]. The upload of
        batch i+1 and the download of batch i-1 run on their own streams while
        batch i is encoded (two device buffers each way), so the copies overlap
        the compute instead of adding to it; each batch's encoder is one CUDA
        graph launch (captured once per batch size and buffer). Returns when
        every copy is done."""
        if len(host_mels) != len(host_feats):
            raise RuntimeError("host_mels and host_feats differ in length")
        if not host_mels:
            return
        dev = self.device
        dm = self.dims
        shape = tuple(host_mels[0].shape)
        if len(shape) != 3 or shape[1] != dm.n_mels or shape[2] != 2 * dm.n_audio_ctx:
            raise RuntimeError("incorrect audio shape")
        feat_shape = (shape[0], dm.n_audio_ctx, dm.n_audio_state)
        for m, f in zip(host_mels, host_feats):
            if m.dtype != torch.int8 or tuple(m.shape) != shape:
                raise RuntimeError("every mel batch must be int8 of the first batch's shape")
            if f.dtype != torch.int8 or tuple(f.shape) != feat_shape:
                raise RuntimeError(f"every feature buffer must be int8 of shape {feat_shape}")
        d_in, d_out, graphs = self._pipe_slots(shape, feat_shape)
        n_graph = self.graph_launches[("encode_batches", shape[0])]
        comp = torch.cuda.current_stream(dev)
        up, down = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
        up.wait_stream(comp)  # nothing starts before the caller's preceding work
        down.wait_stream(comp)
        ev = lambda: torch.cuda.Event()
        in_ready, in_free = [ev(), ev()], [ev(), ev()]
        out_ready, out_free = [ev(), ev()], [ev(), ev()]

        def upload(i):
            s = i % 2
            with torch.cuda.stream(up):
                if i >= 2:
                    up.wait_event(in_free[s])  # batch i-2 no longer reads d_in[s]
                d_in[s].copy_(host_mels[i], non_blocking=True)
                in_ready[s].record(up)

        upload(0)
        for i in range(len(host_mels)):
            s = i % 2
            if i + 1 < len(host_mels):
                upload(i + 1)
            comp.wait_event(in_ready[s])
            if i >= 2:
                comp.wait_event(out_free[s])  # batch i-2's features are downloaded
            graphs[s].replay()
            self.replayed_launches += n_graph
            in_free[s].record(comp)
            out_ready[s].record(comp)
            with torch.cuda.stream(down):
                down.wait_event(out_ready[s])
                host_feats[i].copy_(d_out[s], non_blocking=True)
                out_free[s].record(down)
        comp.wait_stream(down)

    def _block(self, L, ws, B, T, H, d):
        """One encoder block (ResidualAttentionBlock_int.forward without cross
        attention) on the resident INT15 stream ws['x16'] [B*T, d]."""
        M = B * T
        x16, h, qkv, att = ws["x16"], ws["h"], ws["qkv"], ws["att"]
        # Row sums only where a GEMM still has a zero point to apply: the LN
        # then also clears rs_att, which the attention accumulates its output
        # row sums into (the out-projection's zero-point term)
        self._ln(L["attn_ln"], x16, M, h, rowsum_out=_rs(L["qkv"], ws["rs_h"]), rowsum_zero=_rs(L["out"], ws["rs_att"]))
        # with the tensor-core attention, the QKV GEMM writes V directly as V^T
        tc = L["attn"].fb in self._exp_tables
        self._gemm(h, d, M, L["qkv"], qkv, 3 * d, _lib.IW_GEMM_INT8, rowsum=ws["rs_h"],
                   vt=(ws["vt"], 2 * d, T) if tc else None)
        qp = qkv.data_ptr()
        self._attn(L["attn"], B, H, T, T, qp, (3 * d, T * 3 * d, 64), qp + d, (3 * d, T * 3 * d, 64),
                   qp + 2 * d, (3 * d, T * 3 * d, 64), att.data_ptr(), (d, T * d, 64), vt=ws["vt"], vt_ready=tc,
                   rowsum_out=_rs(L["out"], ws["rs_att"]))
        self._gemm(att, d, M, L["out"], x16, d, _lib.IW_GEMM_LINEAR32_RES, rowsum=ws["rs_att"], residual=x16,
                   res_mult=L["attn_res"])
        self._ln(L["mlp_ln"], x16, M, h, rowsum_out=_rs(L["fc1"], ws["rs_h"]), rowsum_zero=_rs(L["fc2"], ws["rs_f1"]))
        self._gemm(h, d, M, L["fc1"], ws["f1"], 4 * d, _lib.IW_GEMM_INT8, rowsum=ws["rs_h"], gelu_tab=L["gelu_tab"],
                   out_rowsum=_rs(L["fc2"], ws["rs_f1"]))
        self._gemm(ws["f1"], 4 * d, M, L["fc2"], x16, d, _lib.IW_GEMM_LINEAR32_RES, rowsum=ws["rs_f1"],
                   residual=x16, res_mult=L["mlp_res"])

    # ------------------------------------------------------------------
    # decoder
    # ------------------------------------------------------------------
    def _dec_workspace(self, B, max_steps):
        key = (B, max_steps)
        if key in self._dec_ws:
            return self._dec_ws[key]
        dm, dev = self.dims, self.device
        d, L, H, Ta, Tcap = dm.n_text_state, dm.n_text_layer, dm.n_text_head, dm.n_audio_ctx, dm.n_text_ctx
        Tp = len(self.tokens_spec["sot_sequence"])
        R = B * Tp  # rows of the widest step (the prefill)
        e8 = lambda *s: torch.empty(*s, dtype=torch.int8, device=dev)
        e32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)
        ws = dict(
            cross=e8(L * 2 * H * B * Ta * 64), selfkv=e8(L * 2 * B * H * Tcap * 64),
            x16=torch.empty(R, d, dtype=torch.int16, device=dev), h=e8(R, d), rs_h=e32(R), qkv=e8(R, 3 * d),
            q=e8(R, d), att=e8(R, d), rs_att=e32(R), f1=e8(R, 4 * d), rs_f1=e32(R),
            logits=e8(B, self.n_vocab_pad), tokens=torch.zeros(B, Tp + max_steps, dtype=torch.int64, device=dev),
            state=torch.zeros(B, 4, dtype=torch.int32, device=dev), next=torch.zeros(B, dtype=torch.int64, device=dev),
            prefill=torch.tensor([self.tokens_spec["sot_sequence"]] * B, dtype=torch.int64, device=dev),
            pos=torch.zeros(1, dtype=torch.int32, device=dev), tk=torch.zeros(1, dtype=torch.int32, device=dev),
            step=torch.zeros(1, dtype=torch.int32, device=dev))
        self._dec_ws[key] = ws
        return ws

    def cross_kv(self, xa: torch.Tensor, rs_xa: torch.Tensor, ws) -> None:
        """K/V of every cross-attention layer from the encoder output in one
        GEMM, stored head-major [L, 2, H, B, n_audio_ctx, 64]."""
        dev = self.tok_emb.device
        if xa.dtype != torch.int8 or xa.dim() != 3 or xa.device != dev or not xa.is_contiguous():
            raise RuntimeError(f"xa must be contiguous int8 features [B, n_audio_ctx, n_audio_state] on {dev}")
        B, Ta, d = xa.shape
        if self.cross_kv_w.wz is not None and (rs_xa is None or rs_xa.dtype != torch.int32 or rs_xa.device != dev
                                               or rs_xa.numel() != B * Ta or not rs_xa.is_contiguous()):
            raise RuntimeError(f"rs_xa must be the contiguous int32 row sums of xa, {B * Ta} of them, on {dev}")
        self._gemm(xa, d, B * Ta, self.cross_kv_w, ws["cross"], 0, _lib.IW_GEMM_INT8, rowsum=rs_xa,
                   headmajor=(Ta, B))

    def _dec_forward(self, ws, B, T, tokens_ptr, tokens_ld_T, pos: int, graph_mode: bool):
        """One TextDecoder_int.forward over T new tokens per utterance, then
        the greedy step. With graph_mode the position is read from the device
        counters (pos/tk) so the launch sequence can be replayed."""
        dm = self.dims
        d, H, Ta, Tcap = dm.n_text_state, dm.n_text_head, dm.n_audio_ctx, dm.n_text_ctx
        st = _stream()
        M = B * T
        x16, h, qkv, q, att = ws["x16"], ws["h"], ws["qkv"], ws["q"], ws["att"]
        pos_dev = ws["pos"].data_ptr() if graph_mode else None
        _lib.check(_lib.LIB.iw_embed_add_requant15_dev(self.tok_emb.data_ptr(), tokens_ptr, self.dec_pe.data_ptr(),
                                                       pos_dev, pos, self.dec_m.data_ptr(), self.dec_s.data_ptr(),
                                                       x16.data_ptr(), B, T, d, self.dec_m.numel(),
                                                       self.dec_s.numel(), st))
        cross = ws["cross"].data_ptr()
        selfkv = ws["selfkv"].data_ptr()
        layer_cross = 2 * H * B * Ta * 64
        layer_self = 2 * B * H * Tcap * 64
        for l, L in enumerate(self.dec_layers):
            # self attention over the cache (model_int.py:713-740, 1120-1129)
            # the LN also clears rs_att, which the attention kernel then
            # accumulates its output row sums into
            self._ln(L["attn_ln"], x16, M, h, rowsum_out=_rs(L["qkv"], ws["rs_h"]),
                     rowsum_zero=_rs(L["out"], ws["rs_att"]))
            kc = selfkv + l * layer_self
            vc = kc + B * H * Tcap * 64
            # Q row-major; K and V appended to the caches by the same GEMM
            self._gemm(h, d, M, L["qkv"], qkv, 3 * d, _lib.IW_GEMM_INT8, rowsum=ws["rs_h"],
                       kv=(kc, vc, d, H, T, Tcap, pos, pos_dev or 0))
            self._attn(L["attn"], B, H, T, pos + T, qkv.data_ptr(), (3 * d, T * 3 * d, 64),
                       kc, (64, H * Tcap * 64, Tcap * 64), vc, (64, H * Tcap * 64, Tcap * 64),
                       att.data_ptr(), (d, T * d, 64), mask_mode=1,
                       Tk_dev=ws["tk"] if graph_mode else None, Tk_cap=Tcap, rowsum_out=_rs(L["out"], ws["rs_att"]))
            self._gemm(att, d, M, L["out"], x16, d, _lib.IW_GEMM_LINEAR32_RES, rowsum=ws["rs_att"], residual=x16,
                       res_mult=L["attn_res"])
            # cross attention over the encoder states (model_int.py:1139-1157)
            self._ln(L["cross_ln"], x16, M, h, rowsum_out=_rs(L["cq"], ws["rs_h"]),
                     rowsum_zero=_rs(L["cout"], ws["rs_att"]))
            self._gemm(h, d, M, L["cq"], q, d, _lib.IW_GEMM_INT8, rowsum=ws["rs_h"])
            ck = cross + l * layer_cross
            cv = ck + H * B * Ta * 64
            self._attn(L["cattn"], B, H, T, Ta, q.data_ptr(), (d, T * d, 64), ck, (64, Ta * 64, B * Ta * 64),
                       cv, (64, Ta * 64, B * Ta * 64), att.data_ptr(), (d, T * d, 64),
                       rowsum_out=_rs(L["cout"], ws["rs_att"]))
            self._gemm(att, d, M, L["cout"], x16, d, _lib.IW_GEMM_LINEAR32_RES, rowsum=ws["rs_att"], residual=x16,
                       res_mult=L["cross_res"])
            # MLP (model_int.py:1160-1171)
            self._ln(L["mlp_ln"], x16, M, h, rowsum_out=_rs(L["fc1"], ws["rs_h"]),
                     rowsum_zero=_rs(L["fc2"], ws["rs_f1"]))
            self._gemm(h, d, M, L["fc1"], ws["f1"], 4 * d, _lib.IW_GEMM_INT8, rowsum=ws["rs_h"],
                       gelu_tab=L["gelu_tab"], out_rowsum=_rs(L["fc2"], ws["rs_f1"]))
            self._gemm(ws["f1"], 4 * d, M, L["fc2"], x16, d, _lib.IW_GEMM_LINEAR32_RES, rowsum=ws["rs_f1"],
                       residual=x16, res_mult=L["mlp_res"])
        # final LN + classifier on the last position of each utterance
        self._ln(self.dec_ln, x16, M, h)
        self._gemm(h.data_ptr() + (T - 1) * d, T * d, B, self.clf, ws["logits"], self.n_vocab_pad,
                   _lib.IW_GEMM_INT8)
        # greedy step on the device
        tk = self.tokens_spec
        g = _lib.GreedyDesc()
        g.logits, g.ld, g.V, g.alpha = ws["logits"].data_ptr(), self.n_vocab_pad, dm.n_vocab, self.logit_alpha
        g.suppress_bits, g.blank, g.n_blank = self.suppress_bits.data_ptr(), self.blank.data_ptr(), self.blank.numel()
        g.eot, g.timestamp_begin, g.no_timestamps = tk["eot"], tk["timestamp_begin"], tk["no_timestamps"]
        g.max_initial_timestamp_index = self.max_initial_timestamp_index
        g.state, g.tokens, g.ld_tok = ws["state"].data_ptr(), ws["tokens"].data_ptr(), ws["tokens"].shape[1]
        g.step_dev, g.next = ws["step"].data_ptr(), ws["next"].data_ptr()
        _lib.check(_lib.LIB.iw_greedy_step(C.byref(g), B, st))
        _lib.check(_lib.LIB.iw_add_i32(ws["step"].data_ptr(), 1, st))
        _lib.check(_lib.LIB.iw_add_i32(ws["pos"].data_ptr(), T, st))
        _lib.check(_lib.LIB.iw_add_i32(ws["tk"].data_ptr(), T, st))

    # precision 0.02 s per audio token; max_initial_timestamp 1.0 s
    # (DecodingTask.__init__, decoding.py:561-570)
    max_initial_timestamp_index = 50

    def decode(self, xa: torch.Tensor, rs_xa: torch.Tensor, sample_len: int, use_graph: bool = True,
               stop_when_done: bool = False) -> torch.Tensor:
        """Greedy decoding (DecodingTask._main_loop with GreedyDecoder,
        decoding.py:684-712) from the SOT sequence for language "en",
        task "transcribe": returns the token matrix [B, 3 + steps] (CUDA).
        Runs exactly ``sample_len`` steps unless ``stop_when_done`` (which
        synchronises once per step, as the reference's loop test does)."""
        B = xa.shape[0]
        ws = self._dec_workspace(B, sample_len)
        sot = self.tokens_spec["sot_sequence"]
        Tp = len(sot)
        ws["tokens"].zero_()
        ws["tokens"][:, :Tp] = torch.tensor(sot, dtype=torch.int64, device=self.device)
        ws["state"].zero_()
        ws["state"][:, 3] = -1
        ws["pos"].zero_()
        ws["tk"].fill_(1)  # key count of the next single-token step is pos + 1
        ws["step"].fill_(Tp)
        self.cross_kv(xa, rs_xa, ws)
        steps = 0
        # prefill: the whole SOT sequence in one forward (offset 0)
        self._dec_forward(ws, B, Tp, ws["prefill"].data_ptr(), Tp, 0, graph_mode=False)
        steps += 1
        pos = Tp
        g = self._graphs.get((B, sample_len)) if use_graph else None
        if use_graph and g is None and sample_len > 1:
            # capture one single-token step; counters live on the device
            st = torch.cuda.Stream()
            st.wait_stream(torch.cuda.current_stream())
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(st):
                # warm the launch path once outside the capture is not needed:
                # every kernel's attributes are set on the prefill above
                with torch.cuda.graph(g, stream=st):
                    self._dec_forward(ws, B, 1, ws["next"].data_ptr(), 1, 0, graph_mode=True)
            torch.cuda.current_stream().wait_stream(st)
            self._graphs[(B, sample_len)] = g
            # capture does not execute: restore nothing
        while steps < sample_len:
            if stop_when_done and bool((ws["state"][:, 1] == self.tokens_spec["eot"]).all()):
                break
            if g is not None:
                g.replay()
            else:
                self._dec_forward(ws, B, 1, ws["next"].data_ptr(), 1, pos, graph_mode=False)
            pos += 1
            steps += 1
        return ws["tokens"][:, :Tp + steps]

    def transcribe_tokens(self, mel_i8: torch.Tensor, sample_len: int, **kw) -> torch.Tensor:
        xa = self.encoder(mel_i8)
        ws = self._enc_ws[mel_i8.shape[0]]
        return self.decode(xa, ws["rs_xa"], sample_len, **kw)
