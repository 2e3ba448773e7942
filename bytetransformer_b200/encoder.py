"""Python host side over the C ABI: torch tensors supply device memory and
streams, every computation goes through libbt_b200.so.

`bert_transformer(...)` mirrors the reference's functional operator
`torch.ops.ByteTransformer.BertTransformer` (bytetransformer/th_op/ths_op_f.cc:28-95):
same argument order, names, defaults and error behaviour (RuntimeError on bad
input).  `Encoder` is the reusable object form (the reference's C++
`BertTransformer<HALF>` used through bytetransformer/th_op/bert_transformer_ext.h:40-118)
extended to a stack of layers.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import List, Optional, Sequence

import torch

from . import _abi

WEIGHT_NAMES = (
    "qkv_kernel", "qkv_bias", "attr_output_kernel", "attr_output_bias",
    "attr_output_layernorm_gamma", "attr_output_layernorm_beta", "inter_kernel", "inter_bias",
    "output_kernel", "output_bias", "output_layernorm_gamma", "output_layernorm_beta")
_LOOSE = {4, 5, 10, 11}  # LayerNorm gamma/beta: dtype not checked by the reference (CHECK_INPUT_LOOSE)


_current_device = torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream_ptr(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class _On:
    """`with torch.cuda.device(device)` that gives the device's current stream, for calls that last microseconds: nothing
    is switched where the device is current already."""
    __slots__ = ("index", "guard")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.guard = None
        if _current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check(t: torch.Tensor, name: str, dtype=None):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"Inconsistency of Tensor type: {name}")


class Encoder:
    """A stack of BERT encoder layers bound to one CUDA device."""

    def __init__(self, head_num: int, head_size: int, layers: Sequence[Sequence[torch.Tensor]], *,
                 max_batch_size: int = 65535, max_seq_len: int = 1024, ln_eps: float = 1e-6,
                 gelu: str = "erf", tao: float = 1.0):
        if not layers:
            raise RuntimeError("at least one layer of weights is required")
        self._lib = _abi.load()
        self.head_num, self.head_size = int(head_num), int(head_size)
        self.hidden = self.head_num * self.head_size
        first = layers[0]
        if len(first) != 12:
            raise RuntimeError("each layer needs 12 weight tensors")
        self.device = first[0].device
        if first[0].dtype != torch.float16:
            raise RuntimeError("only fp16 weights are supported (the fp32 template of the reference "
                               "is not built for sm_100a)")
        gb_fp32 = first[10].dtype == torch.float32  # bert_transformer_ext.h:60-63
        self._layers = []  # keeps the tensors alive: the library stores raw pointers only
        cfg = _abi.bt_config(self.head_num, self.head_size, int(max_batch_size), int(max_seq_len), 4,
                             float(ln_eps), _abi.BT_GELU_ERF if gelu == "erf" else _abi.BT_GELU_TANH,
                             float(tao), int(gb_fp32), self.device.index if self.device.index is not None else -1)
        if gelu not in ("erf", "tanh"):
            raise RuntimeError("gelu must be 'erf' or 'tanh'")
        h = C.c_void_p()
        rc = self._lib.bt_create(C.byref(cfg), C.byref(h))
        if rc != _abi.BT_OK:
            raise _abi.BtError(rc, "bt_create",
                               "head_size must be 64 and the device must be compute capability 10.x")
        self._h = h
        H = self.hidden
        shapes = [(H, 3 * H), (3 * H,), (H, H), (H,), (H,), (H,), (H, 4 * H), (4 * H,), (4 * H, H), (H,), (H,), (H,)]
        for li, w in enumerate(layers):
            if len(w) != 12:
                raise RuntimeError("each layer needs 12 weight tensors")
            for i, t in enumerate(w):
                _check(t, WEIGHT_NAMES[i], None if i in _LOOSE else torch.float16)
                if tuple(t.shape) != shapes[i]:
                    raise RuntimeError(f"{WEIGHT_NAMES[i]} has shape {tuple(t.shape)}, expected {shapes[i]}")
                if i in _LOOSE and t.dtype != (torch.float32 if gb_fp32 else torch.float16):
                    raise RuntimeError("LayerNorm gamma/beta must all be fp16 or all be fp32")
            lw = _abi.bt_layer_weights(*[t.data_ptr() for t in w])
            self._call("bt_set_layer_weights", self._h, li, C.byref(lw))
            self._layers.append(list(w))
        self.n_layers = len(self._layers)
        self._ws: Optional[torch.Tensor] = None

    # ------------------------------------------------------------------ helpers
    def _call(self, name, *args):
        rc = getattr(self._lib, name)(*args)
        if rc != _abi.BT_OK:
            raise _abi.BtError(rc, name, self._lib.bt_last_error(self._h).decode())
        return rc

    def close(self):
        if getattr(self, "_h", None):
            self._lib.bt_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _workspace(self, nbytes: int) -> torch.Tensor:
        if self._ws is None or self._ws.numel() < nbytes:
            self._ws = torch.empty(nbytes, dtype=torch.int8, device=self.device)
        return self._ws

    def device_status(self) -> int:
        st = C.c_int(0)
        self._call("bt_device_status", self._h, _stream_ptr(self.device), C.byref(st))
        return st.value

    def selftest_bounded_wait(self, max_cycles: int, gave_up: torch.Tensor | None = None):
        """Enqueue the library's failure-path self-test: a wait that nothing satisfies gives up after
        about `max_cycles` SM cycles and leaves BT_STATUS_SELFTEST_TIMEOUT in the status word."""
        if gave_up is not None:
            _check(gave_up, "gave_up", torch.int32)
        self._call("bt_selftest_bounded_wait", self._h, int(max_cycles),
                   gave_up.data_ptr() if gave_up is not None else None, _stream_ptr(self.device))

    def profile_enable(self, on: bool = True):
        self._call("bt_profile_enable", self._h, int(bool(on)))

    def profile_read(self):
        """{kind: (milliseconds, launches)} since the last profile_enable(True)."""
        n = len(_abi.PROF_KINDS)
        ms = (C.c_double * n)()
        cnt = (C.c_longlong * n)()
        self._call("bt_profile_read", self._h, ms, cnt)
        return {k: (ms[i], cnt[i]) for i, k in enumerate(_abi.PROF_KINDS)}

    # ----------------------------------------------------------------- forwards
    def _check_io(self, x, attr_mask):
        _check(x, "input", torch.float16)
        _check(attr_mask, "attr_mask", torch.float16)
        if x.dim() != 3 or x.shape[2] != self.hidden:
            raise RuntimeError("input must be [batch, seq_len, head_num*head_size]")
        B, S = int(x.shape[0]), int(x.shape[1])
        if S > 1024:
            raise RuntimeError("Input seq_len too long")  # th_op/util.h:40
        if tuple(attr_mask.shape) != (B, S, S):
            raise RuntimeError("attr_mask must be [batch, seq_len, seq_len]")
        return B, S

    def forward_layer(self, layer: int, x: torch.Tensor, attr_mask: torch.Tensor) -> torch.Tensor:
        """One layer, padded in / padded out, padding rows zero (the reference op)."""
        B, S = self._check_io(x, attr_mask)
        with torch.cuda.device(self.device):
            out = torch.empty_like(x)
            n = C.c_size_t()
            self._call("bt_workspace_bytes", self._h, B, S, C.byref(n))
            ws = self._workspace(n.value)
            self._call("bt_layer_forward_padded", self._h, int(layer), x.data_ptr(), attr_mask.data_ptr(),
                       out.data_ptr(), ws.data_ptr(), ws.numel(), B, S, _stream_ptr(self.device))
        return out

    def forward(self, x: torch.Tensor, attr_mask: torch.Tensor, n_layers: Optional[int] = None) -> torch.Tensor:
        """All layers in one call: pack once, run the stack packed, scatter once."""
        B, S = self._check_io(x, attr_mask)
        nl = self.n_layers if n_layers is None else int(n_layers)
        with torch.cuda.device(self.device):
            out = torch.empty_like(x)
            n = C.c_size_t()
            self._call("bt_workspace_bytes", self._h, B, S, C.byref(n))
            ws = self._workspace(n.value)
            self._call("bt_stack_forward_padded", self._h, nl, x.data_ptr(), attr_mask.data_ptr(), out.data_ptr(),
                       ws.data_ptr(), ws.numel(), B, S, _stream_ptr(self.device))
        return out

    def forward_ids(self, emb: "EmbeddingWeights", token_ids: torch.Tensor, attr_mask: torch.Tensor,
                    type_ids: Optional[torch.Tensor] = None, position_ids: Optional[torch.Tensor] = None,
                    n_layers: Optional[int] = None) -> torch.Tensor:
        """The whole model front to back: embeddings of the valid tokens straight into the packed
        activation, all layers, scatter once (the padded input tensor never exists)."""
        _check(token_ids, "token_ids", torch.int32)
        _check(attr_mask, "attr_mask", torch.float16)
        if token_ids.dim() != 2 or attr_mask.dim() != 3:
            raise RuntimeError("token_ids must be [batch, seq_len], attr_mask [batch, seq_len, seq_len]")
        B, S = int(token_ids.shape[0]), int(token_ids.shape[1])
        if tuple(attr_mask.shape) != (B, S, S):
            raise RuntimeError("attr_mask must be [batch, seq_len, seq_len]")
        for t, n in ((type_ids, "type_ids"), (position_ids, "position_ids")):
            if t is not None:
                _check(t, n, torch.int32)
                if tuple(t.shape) != (B, S):
                    raise RuntimeError(f"{n} must be [batch, seq_len]")
        nl = self.n_layers if n_layers is None else int(n_layers)
        with torch.cuda.device(self.device):
            out = torch.empty(B, S, self.hidden, dtype=torch.float16, device=self.device)
            n = C.c_size_t()
            self._call("bt_workspace_bytes", self._h, B, S, C.byref(n))
            ws = self._workspace(n.value)
            w = emb.as_struct()
            self._call("bt_stack_forward_ids", self._h, nl, C.byref(w), token_ids.data_ptr(),
                       type_ids.data_ptr() if type_ids is not None else None,
                       position_ids.data_ptr() if position_ids is not None else None, attr_mask.data_ptr(),
                       out.data_ptr(), ws.data_ptr(), ws.numel(), B, S, _stream_ptr(self.device))
        return out

    def forward_general(self, x: torch.Tensor, attr_mask: torch.Tensor, attention_bias: Optional[torch.Tensor] = None,
                        n_layers: Optional[int] = None) -> torch.Tensor:
        """All layers with the reference's padded-path attention semantics: nothing is packed, the whole
        [B,S,S] mask is applied element by element as (1 - mask) * -10000 and `attention_bias`
        ([head_num,S,S] fp16, optional) is added to the scaled scores; every output row is computed."""
        B, S = self._check_io(x, attr_mask)
        if attention_bias is not None:
            _check(attention_bias, "attention_bias", torch.float16)
            if tuple(attention_bias.shape) != (self.head_num, S, S):
                raise RuntimeError("attention_bias must be [head_num, seq_len, seq_len]")
        nl = self.n_layers if n_layers is None else int(n_layers)
        with torch.cuda.device(self.device):
            out = torch.empty_like(x)
            n = C.c_size_t()
            self._call("bt_workspace_bytes" if attention_bias is None else "bt_workspace_bytes_bias", self._h, B, S,
                       C.byref(n))
            ws = self._workspace(n.value)
            self._call("bt_stack_forward_padded_general", self._h, nl, x.data_ptr(), attr_mask.data_ptr(),
                       attention_bias.data_ptr() if attention_bias is not None else None, out.data_ptr(),
                       ws.data_ptr(), ws.numel(), B, S, _stream_ptr(self.device))
        return out

    def packed_workspace_bytes(self, batch: int, total_tokens: int) -> int:
        n = C.c_size_t()
        self._call("bt_workspace_bytes_packed", self._h, int(batch), int(total_tokens), C.byref(n))
        return n.value

    def forward_packed(self, x_packed: torch.Tensor, cu_seqlens: torch.Tensor, max_len: int,
                       out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                       n_layers: Optional[int] = None) -> torch.Tensor:
        """Packed in / packed out: x_packed [T,H] fp16, cu_seqlens int32 [B+1] on the device."""
        _check(x_packed, "x_packed", torch.float16)
        _check(cu_seqlens, "cu_seqlens", torch.int32)
        if x_packed.dim() != 2 or x_packed.shape[1] != self.hidden:
            raise RuntimeError("x_packed must be [total_tokens, head_num*head_size]")
        T = int(x_packed.shape[0])
        B = int(cu_seqlens.numel()) - 1
        nl = self.n_layers if n_layers is None else int(n_layers)
        with torch.cuda.device(self.device):
            if out is None:
                out = torch.empty_like(x_packed)
            ws = workspace if workspace is not None else self._workspace(self.packed_workspace_bytes(B, T))
            self._call("bt_stack_forward_packed", self._h, nl, x_packed.data_ptr(), cu_seqlens.data_ptr(), B,
                       int(max_len), T, out.data_ptr(), ws.data_ptr(), ws.numel(), _stream_ptr(self.device))
        return out

    # -------------------------------------------------------- single steps (tests, tools)
    def gemm(self, a: torch.Tensor, w: torch.Tensor, bias=None, residual=None, *, epilogue=_abi.BT_EPI_NONE,
             gelu=_abi.BT_GELU_ERF, m_dev: Optional[torch.Tensor] = None) -> torch.Tensor:
        _check(a, "a", torch.float16)
        _check(w, "w", torch.float16)
        M, K = a.shape
        N = w.shape[1]
        odt = torch.float32 if epilogue == _abi.BT_EPI_BIAS_RESIDUAL_F32OUT else torch.float16
        out = torch.zeros(M, N, dtype=odt, device=a.device)
        self._call("bt_gemm", self._h, a.data_ptr(), w.data_ptr(), out.data_ptr(),
                   bias.data_ptr() if bias is not None else None,
                   residual.data_ptr() if residual is not None else None,
                   m_dev.data_ptr() if m_dev is not None else None, int(M), int(N), int(K), int(epilogue), int(gelu),
                   _stream_ptr(a.device))
        return out

    def gemm_layernorm(self, a, w, bias, residual, gamma, beta, eps=1e-6, m_dev=None) -> torch.Tensor:
        """LayerNorm(a @ w + bias + residual) * gamma + beta in one kernel (bt_gemm_layernorm)."""
        M, K = a.shape
        N = w.shape[1]
        scratch = torch.empty(M, N, dtype=torch.float32, device=a.device)
        out = torch.zeros(M, N, dtype=torch.float16, device=a.device)
        self._call("bt_gemm_layernorm", self._h, a.data_ptr(), w.data_ptr(), bias.data_ptr(), residual.data_ptr(),
                   gamma.data_ptr(), beta.data_ptr(), int(gamma.dtype == torch.float32), float(eps),
                   scratch.data_ptr(), out.data_ptr(), m_dev.data_ptr() if m_dev is not None else None,
                   int(M), int(N), int(K), _stream_ptr(a.device))
        return out

    def attention(self, qkv: torch.Tensor, cu_seqlens: torch.Tensor, max_len: int) -> torch.Tensor:
        _check(qkv, "qkv", torch.float16)
        _check(cu_seqlens, "cu_seqlens", torch.int32)
        rows = int(qkv.shape[0])
        ctx = torch.zeros(rows, self.hidden, dtype=torch.float16, device=qkv.device)
        self._call("bt_attention", self._h, qkv.data_ptr(), ctx.data_ptr(), cu_seqlens.data_ptr(),
                   int(cu_seqlens.numel()) - 1, int(max_len), rows, _stream_ptr(qkv.device))
        return ctx


# ---------------------------------------------------------------------------------------------
# free functions over the stateless entry points
def embedding_layernorm(word_emb: torch.Tensor, pos_emb: torch.Tensor, type_emb: torch.Tensor, gamma: torch.Tensor,
                        beta: torch.Tensor, token_ids: torch.Tensor, type_ids: Optional[torch.Tensor] = None,
                        position_ids: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Encoder input [B,S,H] = LayerNorm(word[token] + position + type) (the step before the stack)."""
    for t, n in ((word_emb, "word_emb"), (pos_emb, "pos_emb"), (type_emb, "type_emb")):
        _check(t, n, torch.float16)
    _check(token_ids, "token_ids", torch.int32)
    if token_ids.dim() != 2:
        raise RuntimeError("token_ids must be [batch, seq_len]")
    gb32 = gamma.dtype == torch.float32
    _check(gamma, "gamma", torch.float32 if gb32 else torch.float16)
    _check(beta, "beta", gamma.dtype)
    B, S = int(token_ids.shape[0]), int(token_ids.shape[1])
    H = int(word_emb.shape[1])
    for t, n in ((type_ids, "type_ids"), (position_ids, "position_ids")):
        if t is not None:
            _check(t, n, torch.int32)
            if tuple(t.shape) != (B, S):
                raise RuntimeError(f"{n} must be [batch, seq_len]")
    lib = _abi.load()
    with torch.cuda.device(word_emb.device):
        out = torch.empty(B, S, H, dtype=torch.float16, device=word_emb.device)
        rc = lib.bt_embedding_layernorm(word_emb.data_ptr(), pos_emb.data_ptr(), type_emb.data_ptr(), gamma.data_ptr(),
                                        beta.data_ptr(), int(gb32), token_ids.data_ptr(),
                                        type_ids.data_ptr() if type_ids is not None else None,
                                        position_ids.data_ptr() if position_ids is not None else None, out.data_ptr(),
                                        B, S, H, int(word_emb.shape[0]), int(pos_emb.shape[0]), int(type_emb.shape[0]),
                                        float(eps), _stream_ptr(word_emb.device))
    if rc != 0:
        raise _abi.BtError(rc, "bt_embedding_layernorm")
    return out


class EmbeddingWeights:
    """Tables and LayerNorm parameters of the embedding front end (fp16 tables, gamma/beta fp16 or fp32)."""

    def __init__(self, word_emb, pos_emb, type_emb, gamma, beta, eps: float = 1e-6):
        for t, n in ((word_emb, "word_emb"), (pos_emb, "pos_emb"), (type_emb, "type_emb")):
            _check(t, n, torch.float16)
        self.gb32 = gamma.dtype == torch.float32
        _check(gamma, "gamma", torch.float32 if self.gb32 else torch.float16)
        _check(beta, "beta", torch.float32 if self.gb32 else torch.float16)
        self.tensors = (word_emb, pos_emb, type_emb, gamma, beta)   # keeps the device memory alive
        self.eps = float(eps)

    def as_struct(self) -> "_abi.bt_embedding_weights":
        w, p, t, g, b = self.tensors
        return _abi.bt_embedding_weights(w.data_ptr(), p.data_ptr(), t.data_ptr(), g.data_ptr(), b.data_ptr(),
                                         1 if self.gb32 else 0, int(w.shape[0]), int(p.shape[0]), int(t.shape[0]), self.eps)


def embedding_layernorm_packed(emb: EmbeddingWeights, token_ids: torch.Tensor, batch_idx: torch.Tensor,
                               word_idx: torch.Tensor, type_ids: Optional[torch.Tensor] = None,
                               position_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Embedding + LayerNorm of the valid tokens only, packed: row r of the result is the token at padded
    position word_idx[r] (offsets from build_offsets); rows from the token count on stay zero."""
    _check(token_ids, "token_ids", torch.int32)
    _check(batch_idx, "batch_idx", torch.int32)
    _check(word_idx, "word_idx", torch.int32)
    B, S = int(token_ids.shape[0]), int(token_ids.shape[1])
    H = int(emb.tensors[0].shape[1])
    out = torch.zeros(B * S, H, dtype=torch.float16, device=token_ids.device)
    w = emb.as_struct()
    rc = _abi.load().bt_embedding_layernorm_packed(
        C.byref(w), token_ids.data_ptr(), type_ids.data_ptr() if type_ids is not None else None,
        position_ids.data_ptr() if position_ids is not None else None, batch_idx.data_ptr(), word_idx.data_ptr(),
        out.data_ptr(), B, S, H, _stream_ptr(token_ids.device))
    if rc != _abi.BT_OK:
        raise RuntimeError(f"bt_embedding_layernorm_packed failed ({_abi.ERROR_NAMES.get(rc, rc)})")
    return out


def pooler(encoder_out: torch.Tensor, W: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """pooled [B,H] = tanh(encoder_out[:,0,:] @ W + bias) (the step after the stack)."""
    _check(encoder_out, "encoder_out", torch.float16)
    _check(W, "W", torch.float16)
    _check(bias, "bias", torch.float16)
    B, S, H = (int(v) for v in encoder_out.shape)
    if tuple(W.shape) != (H, H) or tuple(bias.shape) != (H,):
        raise RuntimeError("W must be [hidden, hidden] and bias [hidden]")
    lib = _abi.load()
    with torch.cuda.device(encoder_out.device):
        out = torch.empty(B, H, dtype=torch.float16, device=encoder_out.device)
        rc = lib.bt_pooler(encoder_out.data_ptr(), W.data_ptr(), bias.data_ptr(), out.data_ptr(), B, S, H,
                           _stream_ptr(encoder_out.device))
    if rc != 0:
        raise _abi.BtError(rc, "bt_pooler")
    return out


def mask_is_right_padded(attr_mask: torch.Tensor) -> bool:
    """True when the packed entry points would honour `attr_mask` [B,S,S] (they look at row 0 only, as the
    reference's prefix-sum kernel does); otherwise use Encoder.forward_general.  Synchronises the stream."""
    _check(attr_mask, "attr_mask", torch.float16)
    if attr_mask.dim() != 3 or attr_mask.shape[1] != attr_mask.shape[2]:
        raise RuntimeError("attr_mask must be [batch, seq_len, seq_len]")
    lib = _abi.load()
    with torch.cuda.device(attr_mask.device):
        scratch = torch.empty(1, dtype=torch.int32, device=attr_mask.device)
        res = C.c_int(0)
        rc = lib.bt_mask_is_right_padded(attr_mask.data_ptr(), int(attr_mask.shape[0]), int(attr_mask.shape[1]),
                                         scratch.data_ptr(), C.byref(res), _stream_ptr(attr_mask.device))
    if rc != 0:
        raise _abi.BtError(rc, "bt_mask_is_right_padded")
    return bool(res.value)


def build_offsets(attr_mask: torch.Tensor):
    """(batch_idx int32[B+1], word_idx int32[B*S]) on the device; only the first
    batch_idx[B] entries of word_idx are defined."""
    lib = _abi.load()
    _check(attr_mask, "attr_mask", torch.float16)
    B, S = int(attr_mask.shape[0]), int(attr_mask.shape[1])
    batch_idx = torch.empty(B + 1, dtype=torch.int32, device=attr_mask.device)
    word_idx = torch.full((B * S,), -1, dtype=torch.int32, device=attr_mask.device)
    rc = lib.bt_build_offsets(attr_mask.data_ptr(), B, S, batch_idx.data_ptr(), word_idx.data_ptr(),
                              _stream_ptr(attr_mask.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_build_offsets")
    return batch_idx, word_idx


def pack_rows(x_padded: torch.Tensor, batch_idx: torch.Tensor, out: Optional[torch.Tensor] = None):
    lib = _abi.load()
    B, S, H = x_padded.shape
    if out is None:
        out = torch.zeros(B * S, H, dtype=torch.float16, device=x_padded.device)
    rc = lib.bt_pack_rows(x_padded.data_ptr(), out.data_ptr(), batch_idx.data_ptr(), None, B, S, H,
                          _stream_ptr(x_padded.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_pack_rows")
    return out


def restore_rows(x_packed: torch.Tensor, batch_idx: torch.Tensor, B: int, S: int):
    lib = _abi.load()
    H = x_packed.shape[1]
    out = torch.full((B, S, H), float("nan"), dtype=torch.float16, device=x_packed.device)
    rc = lib.bt_restore_rows(x_packed.data_ptr(), out.data_ptr(), batch_idx.data_ptr(), B, S, H,
                             _stream_ptr(x_packed.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_restore_rows")
    return out


def add_bias_residual_layernorm(x, bias, residual, gamma, beta, eps=1e-6, m_dev=None):
    lib = _abi.load()
    M, H = x.shape
    out = torch.zeros(M, H, dtype=torch.float16, device=x.device)
    rc = lib.bt_add_bias_residual_layernorm(
        x.data_ptr(), int(x.dtype == torch.float32), bias.data_ptr() if bias is not None else None,
        residual.data_ptr() if residual is not None else None, gamma.data_ptr(), beta.data_ptr(),
        int(gamma.dtype == torch.float32), out.data_ptr(), m_dev.data_ptr() if m_dev is not None else None,
        M, H, float(eps), _stream_ptr(x.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_add_bias_residual_layernorm")
    return out


def add_bias_residual_layernorm_restore(x, bias, residual, gamma, beta, batch_idx, B, S, eps=1e-6):
    lib = _abi.load()
    H = x.shape[1]
    out = torch.full((B, S, H), float("nan"), dtype=torch.float16, device=x.device)
    rc = lib.bt_add_bias_residual_layernorm_restore(
        x.data_ptr(), int(x.dtype == torch.float32), bias.data_ptr() if bias is not None else None,
        residual.data_ptr() if residual is not None else None, gamma.data_ptr(), beta.data_ptr(),
        int(gamma.dtype == torch.float32), out.data_ptr(), batch_idx.data_ptr(), B, S, H, float(eps),
        _stream_ptr(x.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_add_bias_residual_layernorm_restore")
    return out


def add_bias_gelu_(x, bias, gelu="erf"):
    lib = _abi.load()
    M, N = x.shape
    rc = lib.bt_add_bias_gelu(x.data_ptr(), bias.data_ptr(), None, M, N,
                              _abi.BT_GELU_ERF if gelu == "erf" else _abi.BT_GELU_TANH, _stream_ptr(x.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_add_bias_gelu")
    return x


def masked_softmax_(logits, attr_mask, scale=1.0):
    """logits [nh,B,S,S] (the reference's layout), in place."""
    lib = _abi.load()
    nh, B, S, _ = logits.shape
    rc = lib.bt_masked_softmax(logits.data_ptr(), attr_mask.data_ptr(), B, nh, S, float(scale),
                               _stream_ptr(logits.device))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_masked_softmax")
    return logits


_FP32 = {torch.float16: 0, torch.float32: 1}


def _half_or_float(t: torch.Tensor, name: str, device=None) -> int:
    """1 for fp32, 0 for fp16; anything else is refused.  `device`: where the call's other tensors are."""
    _check(t, name)
    if t.dtype not in _FP32:
        raise RuntimeError(f"{name} must be fp16 or fp32")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the other tensors are on {device}")
    return _FP32[t.dtype]


# The library's sizes are 32 bits wide: what does not fit is refused before it is cut off.
_SIZE_LIMIT = 1 << 31
_TOO_LARGE = "sizes must be below 2^31 and not negative"


def _check_distances(buckets, heads, q_len, k_len, max_distance, q_start):
    """Sizes of a bias; those that are added to one another leave room for the sums."""
    if not 0 <= buckets < _SIZE_LIMIT > heads:
        raise RuntimeError(_TOO_LARGE)
    if not (0 <= q_len <= 1 << 29 and 0 <= k_len <= 1 << 29 and -(1 << 29) <= q_start <= 1 << 29 and 0 < max_distance <= 1 << 20):
        raise RuntimeError("lengths and q_start must be at most 2^29, max_distance at most 2^20")


def _relative_bias(table, fp32, buckets, heads, q_len, k_len, max_distance, bidirectional, q_start, out_dtype):
    """The launch of relative_position_bias, whose arguments have been looked at."""
    if q_len == 0 or k_len == 0:
        return torch.empty(heads, q_len, k_len, dtype=out_dtype, device=table.device)
    lib = _abi.load()
    with _On(table.device) as stream:
        out = torch.empty(heads, q_len, k_len, dtype=out_dtype, device=table.device)
        rc = lib.bt_relative_position_bias(table.data_ptr(), fp32, buckets, int(max_distance), int(bool(bidirectional)),
                                           heads, q_len, k_len, int(q_start), out.data_ptr(),
                                           int(out_dtype == torch.float32), stream)
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_relative_position_bias")
    return out


class _RelativeBias(torch.autograd.Function):
    """relative_position_bias of a table that asks for its gradient."""

    @staticmethod
    def forward(ctx, table, *how):
        ctx.table_dtype, ctx.how = table.dtype, how
        return _relative_bias(table, *how)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if torch.cuda.is_current_stream_capturing():
            # autograd itself does not survive a capture that meets leaves of a graph recorded outside it
            raise RuntimeError("the backward pass of relative_position_bias cannot be captured: capture "
                               "relative_position_bias_grad")
        _, buckets, _, _, _, max_distance, bidirectional, q_start, _ = ctx.how
        grad = grad.contiguous()
        if grad.data_ptr() % 16 != 0:  # (part of something larger)
            grad = grad.clone()
        got = relative_position_bias_grad(grad, buckets, max_distance=max_distance, bidirectional=bidirectional,
                                          q_start=q_start)
        return (got.to(ctx.table_dtype),) + (None,) * len(ctx.how)


def relative_position_bias(table: torch.Tensor, q_len: int, k_len: int, *, max_distance: int = 128,
                           bidirectional: bool = True, q_start: int = 0,
                           out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """[heads, q_len, k_len] = table[bucket(k - (q + q_start)), head]: the learned bias by buckets of distance, as
    Encoder.forward_general takes it (fp16) or, with q_len = 1 and out_dtype float32, by distance as window_attention
    does.  table [num_buckets, heads] fp16 or fp32; the buckets are those of bt_relative_position_bias.
    A table that requires its gradient gets it through autograd, by relative_position_bias_grad, in the table's type;
    that backward pass is refused in a stream capture (relative_position_bias_grad itself is not).  The encoder and
    window_attention are forward passes only: what they make of the bias has no history."""
    fp32 = _half_or_float(table, "table")
    if table.dim() != 2:
        raise RuntimeError("table must be [num_buckets, heads]")
    if out_dtype not in (torch.float16, torch.float32):
        raise RuntimeError("out_dtype must be torch.float16 or torch.float32")
    buckets, heads = table.shape
    _check_distances(buckets, heads, q_len, k_len, max_distance, q_start)
    if table.requires_grad and torch.is_grad_enabled():
        return _RelativeBias.apply(table, fp32, buckets, heads, q_len, k_len, max_distance, bidirectional, q_start, out_dtype)
    return _relative_bias(table, fp32, buckets, heads, q_len, k_len, max_distance, bidirectional, q_start, out_dtype)


@functools.lru_cache(maxsize=256)
def _bias_grad_workspace(fp32: int, num_buckets: int, batch: int, heads: int, q_len: int, k_len: int) -> int:
    n = C.c_size_t()
    rc = _abi.load().bt_relative_position_bias_grad_workspace(fp32, num_buckets, batch, heads, q_len, k_len, C.byref(n))
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_relative_position_bias_grad_workspace")
    return n.value


def relative_position_bias_grad(grad: torch.Tensor, num_buckets: int, *, max_distance: int = 128,
                                bidirectional: bool = True, q_start: int = 0) -> torch.Tensor:
    """The gradient of relative_position_bias: [num_buckets, heads] fp32 from that of the bias, [heads, q, k], or of the
    scores of several sequences that one bias was added to, [batch, heads, q, k]; fp16 or fp32."""
    fp32 = _half_or_float(grad, "grad")
    if grad.dim() not in (3, 4):
        raise RuntimeError("grad must be [heads, q_len, k_len] or [batch, heads, q_len, k_len]")
    batch = int(grad.shape[0]) if grad.dim() == 4 else 1
    heads, q_len, k_len = grad.shape[-3:]
    if batch >= _SIZE_LIMIT:
        raise RuntimeError(_TOO_LARGE)
    _check_distances(num_buckets, heads, q_len, k_len, max_distance, q_start)
    if grad.numel() == 0:
        return torch.zeros(num_buckets, heads, dtype=torch.float32, device=grad.device)
    lib = _abi.load()
    n = _bias_grad_workspace(fp32, int(num_buckets), batch, heads, q_len, k_len)
    with _On(grad.device) as stream:
        out = torch.empty(num_buckets, heads, dtype=torch.float32, device=grad.device)
        ws = torch.empty(n, dtype=torch.int8, device=grad.device)
        rc = lib.bt_relative_position_bias_grad(grad.data_ptr(), fp32, int(num_buckets), int(max_distance),
                                                int(bool(bidirectional)), batch, heads, q_len, k_len, int(q_start),
                                                out.data_ptr(), ws.data_ptr(), n, stream)
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_relative_position_bias_grad")
    return out


def _rmsnorm_args(x, residual, gamma, m_dev):
    """(x is fp32, gamma is fp32) of a norm's arguments, which are refused here if they do not fit together."""
    device, shape = x.device, x.shape
    if (m_dev is None and x.is_cuda and x.is_contiguous() and len(shape) == 2 and gamma.shape == shape[1:] and
            gamma.device == device and gamma.is_contiguous() and x.dtype in _FP32 and gamma.dtype in _FP32 and
            (residual is None or (residual.dtype == torch.float16 and residual.shape == shape and
                                  residual.device == device and residual.is_contiguous()))):
        return _FP32[x.dtype], _FP32[gamma.dtype]  # (the usual call; what follows finds out what is wrong, or takes m_dev)
    x_fp32 = _half_or_float(x, "x")
    gamma_fp32 = _half_or_float(gamma, "gamma", x.device)
    if x.dim() != 2 or gamma.dim() != 1 or gamma.shape[0] != x.shape[1]:
        raise RuntimeError("x must be [rows, hidden] and gamma [hidden]")
    if residual is not None:
        _check(residual, "residual", torch.float16)
        if residual.shape != x.shape or residual.device != x.device:
            raise RuntimeError("residual must be fp16 of x's shape, on x's device")
    if m_dev is not None:
        _check(m_dev, "m_dev", torch.int32)
        if m_dev.device != x.device or m_dev.numel() < 1:
            raise RuntimeError("m_dev must be one int32 on x's device")
    return x_fp32, gamma_fp32


def add_residual_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], gamma: torch.Tensor, eps: float = 1e-6,
                         m_dev: Optional[torch.Tensor] = None):
    """(out, sum): sum = x + residual (fp16, the next residual; None without a residual), out = sum / rms(sum) * gamma,
    fp16.  Rows from *m_dev on are left unwritten."""
    x_fp32, gamma_fp32 = _rmsnorm_args(x, residual, gamma, m_dev)
    rows, hidden = x.shape
    if rows >= _SIZE_LIMIT or hidden >= _SIZE_LIMIT:
        raise RuntimeError(_TOO_LARGE)
    lib = _abi.load()
    with _On(x.device) as stream:
        out = torch.empty(rows, hidden, dtype=torch.float16, device=x.device)
        total = torch.empty_like(out) if residual is not None else None
        if rows == 0:
            return out, total
        rc = lib.bt_add_residual_rmsnorm(x.data_ptr(), x_fp32, residual.data_ptr() if residual is not None else None,
                                         gamma.data_ptr(), gamma_fp32, total.data_ptr() if total is not None else None,
                                         out.data_ptr(), m_dev.data_ptr() if m_dev is not None else None, rows, hidden,
                                         eps, stream)
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_add_residual_rmsnorm")
    return out, total


def add_residual_rmsnorm_e4m3(x: torch.Tensor, residual: Optional[torch.Tensor], gamma: torch.Tensor, eps: float = 1e-6,
                              group: int = 0, m_dev: Optional[torch.Tensor] = None):
    """(out, scales, sum): add_residual_rmsnorm with the result in 8 bits, out float8_e4m3fn and fp32 scales with
    out * scales = the norm: one to a row ([rows, 1], group = 0) or to 128 columns ([rows, ceil(hidden/128)], group = 128)."""
    x_fp32, gamma_fp32 = _rmsnorm_args(x, residual, gamma, m_dev)
    if group not in (0, 128):
        raise RuntimeError("group must be 0 (a scale per row) or 128 (a scale per 128 columns)")
    rows, hidden = x.shape
    if rows >= _SIZE_LIMIT or hidden >= _SIZE_LIMIT:
        raise RuntimeError(_TOO_LARGE)
    lib = _abi.load()
    with _On(x.device) as stream:
        out = torch.empty(rows, hidden, dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty(rows, (hidden + 127) // 128 if group else 1, dtype=torch.float32, device=x.device)
        total = torch.empty(rows, hidden, dtype=torch.float16, device=x.device) if residual is not None else None
        if rows == 0:
            return out, scales, total
        rc = lib.bt_add_residual_rmsnorm_e4m3(x.data_ptr(), x_fp32, residual.data_ptr() if residual is not None else None,
                                              gamma.data_ptr(), gamma_fp32,
                                              total.data_ptr() if total is not None else None, out.data_ptr(),
                                              scales.data_ptr(), group, m_dev.data_ptr() if m_dev is not None else None,
                                              rows, hidden, eps, stream)
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_add_residual_rmsnorm_e4m3")
    return out, scales, total


def _rows(t: torch.Tensor, name: str, device) -> int:
    """Heads of a matrix [rows, heads * 64] whose rows may be further apart than they are long."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float16:
        raise RuntimeError(f"Inconsistency of Tensor type: {name}")
    cols = t.shape[1] if t.dim() == 2 else 0
    if cols == 0 or cols % 64 != 0 or t.stride(1) != 1:
        raise RuntimeError(f"{name} must be [rows, heads*64] with contiguous rows")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the other tensors are on {device}")
    return cols // 64


def _ints(t: torch.Tensor, name: str, device) -> int:
    if t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != 1 or t.device != device:
        raise RuntimeError(f"{name} must be a contiguous int32 vector on the device of the other tensors")
    return t.shape[0]


@functools.lru_cache(maxsize=256)
def _window_workspace(batch: int, heads: int, kv_heads: int, max_q_len: int, max_k_len: int, left: int, sinks: int) -> int:
    """Bytes, or 0 where the arguments are such that the call itself will refuse them."""
    n = C.c_size_t()
    rc = _abi.load().bt_window_attention_workspace(batch, heads, kv_heads, max_q_len, max_k_len, left, sinks, C.byref(n))
    return n.value if rc == _abi.BT_OK else 0


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
                     max_q_len: int, max_k_len: int, *, left: int = -1, right: int = -1, sinks: int = 0,
                     k_lens: Optional[torch.Tensor] = None, distance_bias: Optional[torch.Tensor] = None,
                     bias_left: int = 0, scale: float = 0.125, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[rows, heads*64]: packed attention in which a query sees `left` keys before it, `right` behind it and the first
    `sinks` ones of its sequence (bt_window_attention has the definition).  q [rows, heads*64], k and v
    [k_rows, kv_heads*64], fp16, views into a packed QKV product among them; queries are the last ones of their
    sequence's keys, so a single new token over a cache is a sequence of one query (k_lens: how much of each
    sequence's place in the cache is filled).  distance_bias [heads, n] fp32, value of distance j - p at bias_left + j - p.
    Rows that belong to no sequence are left as `out` has them (undefined without `out`)."""
    device = q.device
    heads, kv_heads = _rows(q, "q", device), _rows(k, "k", device)
    rows, k_rows = q.shape[0], k.shape[0]
    if v.shape != k.shape:
        raise RuntimeError("k and v must have the same shape")
    if v.dtype != torch.float16 or v.device != device or v.stride(1) != 1:
        _rows(v, "v", device)  # (says what is wrong)
    batch = _ints(q_offsets, "q_offsets", device) - 1
    if batch < 0 or k_offsets is not q_offsets and _ints(k_offsets, "k_offsets", device) != batch + 1:
        raise RuntimeError("q_offsets and k_offsets must have batch + 1 elements")
    if k_lens is not None and _ints(k_lens, "k_lens", device) != batch:
        raise RuntimeError("k_lens must have batch elements")
    n_bias = 0
    if distance_bias is not None:
        _check(distance_bias, "distance_bias", torch.float32)
        if distance_bias.dim() != 2 or distance_bias.shape[0] != heads or distance_bias.device != device:
            raise RuntimeError("distance_bias must be [heads, n] on the device of the other tensors")
        n_bias = distance_bias.shape[1]
        if not 0 <= bias_left < n_bias:
            raise RuntimeError("bias_left must be a place in distance_bias")
    if out is not None and (_rows(out, "out", device) != heads or out.shape[0] != rows):
        raise RuntimeError("out must have q's shape")
    if not (0 <= max_q_len < 1 << 30 and 0 <= max_k_len < 1 << 30 and sinks >= 0):
        raise RuntimeError("max_q_len and max_k_len must be below 2^30, they and sinks not negative")
    if batch >= _SIZE_LIMIT or rows >= _SIZE_LIMIT or k_rows >= _SIZE_LIMIT or heads >= _SIZE_LIMIT or n_bias >= _SIZE_LIMIT:
        raise RuntimeError(_TOO_LARGE)
    # bounds that no distance reaches, however large, are none (the library's are 32 bits wide)
    left = -1 if left < 0 or left >= max_k_len else left
    right = -1 if right < 0 or right >= 1 << 30 else right
    sinks = min(sinks, max_k_len)
    lib = _abi.load()
    with _On(device) as stream:
        if out is None:
            out = torch.empty(rows, heads * 64, dtype=torch.float16, device=device)
        if rows == 0 or batch == 0 or max_q_len == 0:
            return out
        ws, n = None, 0
        if max_q_len * heads <= 16 * kv_heads:  # few queries: the keys may be cut into ranges
            n = _window_workspace(batch, heads, kv_heads, max_q_len, max_k_len, left, sinks)
            if n:
                ws = torch.empty(n, dtype=torch.int8, device=device)
        # elements from a row to the next; the stride of a single row says nothing, whatever it is
        q_row, out_row = (q.stride(0), out.stride(0)) if rows > 1 else (heads * 64, heads * 64)
        k_row, v_row = (k.stride(0), v.stride(0)) if k_rows > 1 else (kv_heads * 64, kv_heads * 64)
        a = _abi.bt_window_attention_args(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), q_row, k_row, v_row, out_row,
            q_offsets.data_ptr(), k_offsets.data_ptr(), k_lens.data_ptr() if k_lens is not None else None,
            batch, heads, kv_heads, rows, k_rows, max_q_len, max_k_len, left, right, sinks, scale,
            distance_bias.data_ptr() if distance_bias is not None else None, n_bias, bias_left if n_bias else 0,
            ws.data_ptr() if n else None, n)
        rc = lib.bt_window_attention(C.byref(a), stream)
    if rc != _abi.BT_OK:
        raise _abi.BtError(rc, "bt_window_attention")
    return out


def bert_transformer(head_num: int, head_size: int,
                     qkv_kernel, qkv_bias, attr_output_kernel, attr_output_bias,
                     attr_output_layernorm_gamma, attr_output_layernorm_beta,
                     inter_kernel, inter_bias, output_kernel, output_bias,
                     output_layernorm_gamma, output_layernorm_beta,
                     input, attr_mask, is_remove_padding: bool = True,
                     use_fused_attention: bool = True, *, ln_eps: float = 1e-6, gelu: str = "erf"):
    """Drop-in for `torch.ops.ByteTransformer.BertTransformer` (ths_op_f.cc:85-95).

    is_remove_padding=True: the packed path (lengths = valid keys of mask row 0, right padding, padding rows
    of the output zero).  False: the reference's padded semantics (nothing packed, the whole [B,S,S] mask
    applied element by element, every output row computed), which is what a causal or block-diagonal mask
    needs.  `use_fused_attention` is accepted for signature compatibility: attention is fused on both paths.
    The encoder object is built per call, as the reference does (bert_transformer_ext.h:86-110)."""
    w = [qkv_kernel, qkv_bias, attr_output_kernel, attr_output_bias, attr_output_layernorm_gamma,
         attr_output_layernorm_beta, inter_kernel, inter_bias, output_kernel, output_bias,
         output_layernorm_gamma, output_layernorm_beta]
    enc = Encoder(head_num, head_size, [w], ln_eps=ln_eps, gelu=gelu)
    try:
        if not is_remove_padding:
            return enc.forward_general(input, attr_mask, n_layers=1)
        return enc.forward_layer(0, input, attr_mask)
    finally:
        enc.close()
