"""Torch-facing wrappers of libcbx_ops, named after the engine's layer helpers.

Each function takes CUDA tensors (the device memory), enqueues one kernel of
libcbx_ops on the current torch CUDA stream through the C ABI, and returns the
output tensor.  The names and argument meanings follow the chatterbox-cpp
helpers they replace:

  embed_gather_add   t3.cpp:432-455      get_rows x2 + cast + concat + add
  t3_embed_sequence  t3.cpp:428-455      [cond ; speech[prompt] ; tokens] + pos
  add_layernorm      t3.cpp:528-532      residual add, norm, mul(w), add(b)
  layer_norm         cfm_decoder.cpp:29  layer_norm(ctx, x, w, b, eps)
  layernorm_channels cfm_decoder.cpp:144-148  LN over C, mish, * mask
  gelu / silu / mish t3.cpp:537, cfm_decoder.cpp:466, cfm_decoder.cpp:36
  gelu_erf           cfm_decoder.cpp:239, s3enc.cpp:177
  bias_act           t3.cpp:536-537 (fc bias + GELU), cfm_decoder.cpp:114,
                     hift_vocoder.cpp:575 (ELU), :686 / :748 (LeakyReLU)
  sum3_scale         hift_vocoder.cpp:733-739 (ResBlock average)
  sinusoidal_pos_emb cfm_decoder.cpp:49-62 (batched, on the device)
  snake              hift_vocoder.cpp:64-73
  qkv_kv_append_paged  t3.cpp:465-489 on a paged KV cache
  paged_plan, paged_decode_attention, token_logprobs: the rest of a paged decode
                     step (block tables and slots, attention, the answer's log
                     probabilities); the engine decodes one slab per stream

There is no CPU path: inputs must be CUDA tensors and the shared library must
be present, otherwise these raise.
"""
from __future__ import annotations

import ctypes
import functools
import inspect
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from ._lib import (ACT_ELU, ACT_GELU_ERF, ACT_GELU_TANH, ACT_LEAKY_RELU, ACT_MISH, ACT_NONE,
                   ACT_SILU, BCT, BF16, BIAS_NE0, BIAS_NE1, BTC, F16, F32)

_TORCH_TO_CBX = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_ACTS = {None: ACT_NONE, "none": ACT_NONE, "mish": ACT_MISH, "silu": ACT_SILU,
         "gelu": ACT_GELU_TANH, "gelu_tanh": ACT_GELU_TANH, "gelu_erf": ACT_GELU_ERF,
         "leaky_relu": ACT_LEAKY_RELU, "elu": ACT_ELU}
_LAYOUTS = {"BCT": BCT, "BTC": BTC}


def _cbx_type(t: torch.Tensor) -> int:
    try:
        return _TORCH_TO_CBX[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype} (f32, f16, bf16)") from None


def _on_tensor_device(fn):
    """Run a wrapper with its first tensor's device current.  The library
    takes its per-device state (SM count, occupancy, error word) from the
    current device, and the stream comes from the tensor's device, so the two
    must agree; the switch is skipped when they already do."""
    @functools.wraps(fn)
    def wrapper(*args, **kw):
        t = args[0] if args else next(iter(kw.values()), None)
        if (isinstance(t, torch.Tensor) and t.is_cuda
                and t.device.index != torch.cuda.current_device()):
            with torch.cuda.device(t.device):
                return fn(*args, **kw)
        return fn(*args, **kw)
    return wrapper


def _dev(t: torch.Tensor | None, name: str, dtype=None):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (libcbx_ops has no CPU path)")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the call runs on "
                         f"cuda:{torch.cuda.current_device()}: all tensors of a call must "
                         "share its device")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    return ctypes.c_void_p(t.data_ptr())


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _act(act) -> int:
    if isinstance(act, int):
        return act
    try:
        return _ACTS[act]
    except KeyError:
        raise ValueError(f"unknown act {act!r}") from None


def _layout(layout) -> int:
    if isinstance(layout, int):
        return layout
    try:
        return _LAYOUTS[layout]
    except KeyError:
        raise ValueError(f"unknown layout {layout!r} (BCT or BTC)") from None


# ------------------------------------------------------------------ gather --

@_on_tensor_device
def embed_gather_add(tok_table: torch.Tensor, ids: torch.Tensor,
                     pos_table: torch.Tensor | None = None, pos_ids: torch.Tensor | None = None,
                     n_past: int = 0, out_dtype: torch.dtype = torch.float32,
                     err_word: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """out[i] = tok_table[ids[i]] + pos_table[pos_ids[i] or n_past + i] (t3.cpp:440-455)."""
    if ids.dtype != torch.int32:
        raise TypeError("ids must be int32")
    n_rows, hidden = ids.numel(), tok_table.shape[-1]
    if out is None:
        out = torch.empty((n_rows, hidden), dtype=out_dtype, device=ids.device)
    _lib.call("cbx_embed_gather_add", _dev(tok_table, "tok_table"), _cbx_type(tok_table),
              tok_table.shape[0], _dev(pos_table, "pos_table"),
              _cbx_type(pos_table) if pos_table is not None else F32,
              pos_table.shape[0] if pos_table is not None else 0, _dev(ids, "ids"),
              _dev(pos_ids, "pos_ids", torch.int32), int(n_past), n_rows, hidden,
              _dev(out, "out"), _cbx_type(out), _dev(err_word, "err_word", torch.int32),
              _stream(ids))
    return out


@_on_tensor_device
def embed_gather_add_batched(tok_table: torch.Tensor, ids: torch.Tensor,
                             pos_table: torch.Tensor | None = None, n_past: int = 0,
                             out_dtype: torch.dtype = torch.float32,
                             err_word: torch.Tensor | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """A batch of utterances at the same positions: ids [B, T] ->
    out[b, t] = tok_table[ids[b, t]] + pos_table[n_past + t] (t3.cpp:440-455
    per utterance, one launch for the batch).  Returns [B, T, hidden]."""
    if ids.dtype != torch.int32:
        raise TypeError("ids must be int32")
    if ids.dim() != 2:
        raise ValueError(f"ids must be [n_batch, seq_len], got shape {tuple(ids.shape)}")
    n_batch, seq_len = ids.shape
    hidden = tok_table.shape[-1]
    if pos_table is not None and pos_table.shape[-1] != hidden:
        raise ValueError("pos_table and tok_table differ in hidden size")
    if out is None:
        out = torch.empty((n_batch, seq_len, hidden), dtype=out_dtype, device=ids.device)
    elif out.numel() != n_batch * seq_len * hidden:
        raise ValueError(f"out holds {out.numel()} values, needs {n_batch * seq_len * hidden}")
    _lib.call("cbx_embed_gather_add_batched", _dev(tok_table, "tok_table"), _cbx_type(tok_table),
              tok_table.shape[0], _dev(pos_table, "pos_table"),
              _cbx_type(pos_table) if pos_table is not None else F32,
              pos_table.shape[0] if pos_table is not None else 0, _dev(ids, "ids"),
              n_batch, seq_len, int(n_past), hidden, _dev(out, "out"), _cbx_type(out),
              _dev(err_word, "err_word", torch.int32), _stream(ids))
    return out


@_on_tensor_device
def t3_embed_sequence(tok_table: torch.Tensor, tok_ids: torch.Tensor,
                      pos_table: torch.Tensor | None = None, n_past: int = 0,
                      cond: torch.Tensor | None = None, prompt_table: torch.Tensor | None = None,
                      prompt_ids: torch.Tensor | None = None,
                      out_dtype: torch.dtype = torch.float32,
                      err_word: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """The T3 prefill input sequence (t3.cpp:428-455) in one pass:
    [cond rows (f32 [n_cond, H]) ; prompt_table[prompt_ids] ; tok_table[tok_ids]]
    + pos_table[n_past + i].  Returns [n_cond + n_prompt + n_tok, H]."""
    for name, t in (("tok_ids", tok_ids), ("prompt_ids", prompt_ids)):
        if t is not None and t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
    if (prompt_ids is None) != (prompt_table is None):
        raise ValueError("prompt_table and prompt_ids go together")
    hidden = tok_table.shape[-1]
    n_cond = 0 if cond is None else cond.reshape(-1, hidden).shape[0]
    if cond is not None and cond.numel() != n_cond * hidden:
        raise ValueError(f"cond holds {cond.numel()} values, not a multiple of hidden {hidden}")
    n_prompt = 0 if prompt_ids is None else prompt_ids.numel()
    if prompt_table is not None and prompt_table.shape[-1] != hidden:
        raise ValueError("prompt_table and tok_table differ in hidden size")
    n_tok = tok_ids.numel()
    if out is None:
        out = torch.empty((n_cond + n_prompt + n_tok, hidden), dtype=out_dtype,
                          device=tok_table.device)
    _lib.call("cbx_t3_embed_sequence", _dev(cond, "cond", torch.float32), n_cond,
              _dev(prompt_table, "prompt_table"),
              _cbx_type(prompt_table) if prompt_table is not None else F32,
              prompt_table.shape[0] if prompt_table is not None else 0,
              _dev(prompt_ids, "prompt_ids"), n_prompt,
              _dev(tok_table, "tok_table"), _cbx_type(tok_table), tok_table.shape[0],
              _dev(tok_ids, "tok_ids"), n_tok, _dev(pos_table, "pos_table"),
              _cbx_type(pos_table) if pos_table is not None else F32,
              pos_table.shape[0] if pos_table is not None else 0, int(n_past), hidden,
              _dev(out, "out"), _cbx_type(out), _dev(err_word, "err_word", torch.int32),
              _stream(tok_table))
    return out


@_on_tensor_device
def t3_embed_sequence_batched(tok_table: torch.Tensor, tok_ids: torch.Tensor,
                              pos_table: torch.Tensor | None = None, n_past: int = 0,
                              cond: torch.Tensor | None = None,
                              prompt_table: torch.Tensor | None = None,
                              prompt_ids: torch.Tensor | None = None,
                              out_dtype: torch.dtype = torch.float32,
                              err_word: torch.Tensor | None = None,
                              out: torch.Tensor | None = None) -> torch.Tensor:
    """t3_embed_sequence for a batch of utterances in one launch: tok_ids
    [B, n_tok], prompt_ids [B, n_prompt], cond [B, n_cond, H] (or [B, H]).
    Returns [B, n_cond + n_prompt + n_tok, H]."""
    for name, t in (("tok_ids", tok_ids), ("prompt_ids", prompt_ids)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != 2):
            raise TypeError(f"{name} must be an int32 [n_batch, n] tensor")
    if (prompt_ids is None) != (prompt_table is None):
        raise ValueError("prompt_table and prompt_ids go together")
    B, n_tok = tok_ids.shape
    hidden = tok_table.shape[-1]
    n_prompt = 0 if prompt_ids is None else prompt_ids.shape[1]
    if prompt_ids is not None and prompt_ids.shape[0] != B:
        raise ValueError("prompt_ids and tok_ids differ in batch size")
    if prompt_table is not None and prompt_table.shape[-1] != hidden:
        raise ValueError("prompt_table and tok_table differ in hidden size")
    n_cond = 0
    if cond is not None and B * hidden > 0:
        if cond.numel() % (B * hidden):
            raise ValueError(f"cond holds {cond.numel()} values, not a multiple of B * hidden")
        n_cond = cond.numel() // (B * hidden)
    n = n_cond + n_prompt + n_tok
    if out is None:
        out = torch.empty((B, n, hidden), dtype=out_dtype, device=tok_table.device)
    elif out.numel() != B * n * hidden:
        raise ValueError(f"out holds {out.numel()} values, needs {B * n * hidden}")
    _lib.call("cbx_t3_embed_sequence_batched", _dev(cond, "cond", torch.float32), n_cond,
              _dev(prompt_table, "prompt_table"),
              _cbx_type(prompt_table) if prompt_table is not None else F32,
              prompt_table.shape[0] if prompt_table is not None else 0,
              _dev(prompt_ids, "prompt_ids"), n_prompt,
              _dev(tok_table, "tok_table"), _cbx_type(tok_table), tok_table.shape[0],
              _dev(tok_ids, "tok_ids"), n_tok, _dev(pos_table, "pos_table"),
              _cbx_type(pos_table) if pos_table is not None else F32,
              pos_table.shape[0] if pos_table is not None else 0, int(n_past), hidden, B,
              _dev(out, "out"), _cbx_type(out), _dev(err_word, "err_word", torch.int32),
              _stream(tok_table))
    return out


# --------------------------------------------------------------- layernorm --

@_on_tensor_device
def add_layernorm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None,
                  bias: torch.Tensor | None, eps: float = 1e-5, out_dtype=None,
                  return_sum: bool = False, out: torch.Tensor | None = None,
                  sum_out: torch.Tensor | None = None):
    """y = LN(x + residual) * weight + bias over the last dim (t3.cpp:528-532).

    Returns y, or (y, s) with s = x + residual in x's dtype when return_sum."""
    hidden = x.shape[-1]
    n_rows = x.numel() // hidden if hidden else 0
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    if return_sum and sum_out is None:
        sum_out = torch.empty_like(x)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must match x in shape and dtype")
    _lib.call("cbx_add_layernorm", _dev(x, "x"), _dev(residual, "residual"), _cbx_type(x), 0,
              _dev(weight, "weight", torch.float32), _dev(bias, "bias", torch.float32),
              float(eps), n_rows, hidden, _dev(sum_out, "sum_out"), _dev(out, "out"),
              _cbx_type(out), 0, _stream(x))
    return (out, sum_out) if return_sum else out


@_on_tensor_device
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
               eps: float = 1e-5) -> torch.Tensor:
    """layer_norm(ctx, x, w, b, eps) of cfm_decoder.cpp:29-33 / flow_encoder.cpp:58-62."""
    return add_layernorm(x, None, weight, bias, eps)


@_on_tensor_device
def layernorm_channels(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None,
                       eps: float = 1e-5, mask: torch.Tensor | None = None, layout="BCT",
                       act="mish", out: torch.Tensor | None = None) -> torch.Tensor:
    """CausalBlock1D tail act(LN_C(x) * w + b) * mask (cfm_decoder.cpp:144-148).

    x: f32 [B, C, T] (layout "BCT") or [B, T, C] ("BTC"); mask: f32 [B, T]."""
    lay = _layout(layout)
    if x.dim() != 3:
        raise ValueError("x must be 3-D")
    B, C, T = (x.shape[0], x.shape[1], x.shape[2]) if lay == BCT else (x.shape[0], x.shape[2],
                                                                       x.shape[1])
    if out is None:
        out = torch.empty_like(x)
    _lib.call("cbx_layernorm_channels", _dev(x, "x", torch.float32),
              _dev(weight, "weight", torch.float32), _dev(bias, "bias", torch.float32),
              float(eps), _dev(mask, "mask", torch.float32), B, C, T, lay, _act(act),
              _dev(out, "out", torch.float32), _stream(x))
    return out


@_on_tensor_device
def causal_block1d_tail(x: torch.Tensor, conv_bias: torch.Tensor | None,
                        weight: torch.Tensor | None, bias: torch.Tensor | None,
                        eps: float = 1e-5, mask: torch.Tensor | None = None, act="mish",
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """The causal conv's epilogue and the CausalBlock1D tail in one pass
    (cfm_decoder.cpp:114-115, :144-148): act(LN_C(x + conv_bias) * w + b) * mask.

    x: f32 [B, C, T] (the conv GEMM's output); returns f32 [B, T, C] (the
    engine's (C, T) layout); mask: f32 [B, T]."""
    if x.dim() != 3:
        raise ValueError("x must be 3-D")
    B, C, T = x.shape
    if out is None:
        out = torch.empty(B, T, C, dtype=torch.float32, device=x.device)
    if tuple(out.shape) != (B, T, C):
        raise ValueError("out must be [B, T, C]")
    _lib.call("cbx_causal_block1d_tail", _dev(x, "x", torch.float32),
              _dev(conv_bias, "conv_bias", torch.float32), _dev(weight, "weight", torch.float32),
              _dev(bias, "bias", torch.float32), float(eps), _dev(mask, "mask", torch.float32),
              B, C, T, _act(act), _dev(out, "out", torch.float32), _stream(x))
    return out


# -------------------------------------------------------------- activations --

def _unary(fn: str, x: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        out = torch.empty_like(x)
    if out.dtype != x.dtype or out.numel() != x.numel():
        raise ValueError("out must match x")
    _lib.call(fn, _dev(x, "x"), _dev(out, "out"), x.numel(), _cbx_type(x), _stream(x))
    return out


@_on_tensor_device
def gelu(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """ggml_gelu (GELU-tanh) of t3.cpp:537."""
    return _unary("cbx_gelu_tanh", x, out)


@_on_tensor_device
def silu(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """ggml_silu of cfm_decoder.cpp:466 / flow_encoder.cpp:402."""
    return _unary("cbx_silu", x, out)


@_on_tensor_device
def mish(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """mish() of cfm_decoder.cpp:36-38."""
    return _unary("cbx_mish", x, out)


@_on_tensor_device
def gelu_erf(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """ggml_gelu_erf (exact GELU) of cfm_decoder.cpp:239 / s3enc.cpp:177."""
    return _unary("cbx_gelu_erf", x, out)


# ----------------------------------------------------- epilogue neighbours --

@_on_tensor_device
def bias_act(x: torch.Tensor, bias: torch.Tensor | None = None, act=None, axis: str = "ne0",
             act_param: float = 0.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = act(x + bias) over rows of x.shape[-1] elements.

    axis "ne0": bias[j] along the last dim (t3.cpp:536-537 fc bias + GELU);
    axis "ne1": bias[row % len(bias)] per row (conv bias on (T, C),
    cfm_decoder.cpp:114).  act: None, "gelu", "gelu_erf", "silu", "mish",
    "elu", "leaky_relu" (slope act_param; hift_vocoder.cpp:686, :748)."""
    hidden = x.shape[-1]
    n_rows = x.numel() // hidden if hidden else 0
    ax = {"ne0": BIAS_NE0, "ne1": BIAS_NE1}[axis]
    if out is None:
        out = torch.empty_like(x)
    if out.dtype != x.dtype or out.numel() != x.numel():
        raise ValueError("out must match x")
    _lib.call("cbx_bias_act", _dev(x, "x"), _dev(out, "out"), _cbx_type(x), n_rows, hidden,
              _dev(bias, "bias", torch.float32), ax,
              bias.numel() if bias is not None else 0, _act(act), float(act_param), _stream(x))
    return out


@_on_tensor_device
def sum3_scale(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, scale: float = 1.0 / 3.0,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """((a + b) + c) * scale: HiFT's three-ResBlock average (hift_vocoder.cpp:733-739)."""
    if not (a.shape == b.shape == c.shape and a.dtype == b.dtype == c.dtype):
        raise ValueError("a, b, c must match")
    if out is None:
        out = torch.empty_like(a)
    _lib.call("cbx_sum3_scale", _dev(a, "a"), _dev(b, "b"), _dev(c, "c"), float(scale),
              _dev(out, "out"), a.numel(), _cbx_type(a), _stream(a))
    return out


# --------------------------------------------------------------- timesteps --

def sinusoid_freqs(dim: int) -> np.ndarray:
    """Host frequency table of cfm_decoder.cpp:52-56 (f32 [dim // 2])."""
    out = np.empty(dim // 2, np.float32)
    _lib.call("cbx_sinusoid_freqs", int(dim), out.ctypes.data_as(ctypes.c_void_p))
    return out


@_on_tensor_device
def sinusoidal_pos_emb(t: torch.Tensor, dim: int = 320, scale: float = 1000.0, act=None,
                       freqs: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """[n_t, dim] = [sin(a), cos(a)], a = (scale t) freq (cfm_decoder.cpp:49-62), + SiLU."""
    if freqs is None:
        freqs = torch.from_numpy(sinusoid_freqs(dim)).to(t.device)
    n_t = t.numel()
    if out is None:
        out = torch.empty((n_t, dim), dtype=torch.float32, device=t.device)
    _lib.call("cbx_timestep_embed", _dev(t, "t", torch.float32), n_t,
              _dev(freqs, "freqs", torch.float32), int(dim), float(scale), _act(act),
              _dev(out, "out", torch.float32), _stream(t))
    return out


# ------------------------------------------------------------------- snake --

def snake_alpha_inv(alpha: np.ndarray, eps: float = 1e-9) -> np.ndarray:
    """Host 1 / (alpha + eps) in f32 (hift_vocoder.cpp:419-420)."""
    a = np.ascontiguousarray(alpha, np.float32)
    inv = np.empty_like(a)
    _lib.call("cbx_snake_alpha_inv", a.ctypes.data_as(ctypes.c_void_p), a.size, float(eps),
              inv.ctypes.data_as(ctypes.c_void_p))
    return inv


@_on_tensor_device
def snake(x: torch.Tensor, alpha: torch.Tensor, alpha_inv: torch.Tensor | None = None,
          eps: float = 1e-9, layout="BCT", out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x + sin^2(alpha x) * alpha_inv (hift_vocoder.cpp:64-73).

    x: f32 [B, C, T] ("BCT") or [B, T, C] ("BTC"); alpha, alpha_inv: f32 [C]."""
    lay = _layout(layout)
    shape = x.shape
    x3 = x.unsqueeze(0) if x.dim() == 2 else x          # [C, T] / [T, C] -> one item
    if x3.dim() != 3:
        raise ValueError("x must be 2-D or 3-D")
    B, C, T = (x3.shape[0], x3.shape[1], x3.shape[2]) if lay == BCT else (
        x3.shape[0], x3.shape[2], x3.shape[1])
    if out is None:
        out = torch.empty_like(x)
    if out.shape != shape:
        raise ValueError("out must match x")
    _lib.call("cbx_snake", _dev(x, "x", torch.float32), _dev(alpha, "alpha", torch.float32),
              _dev(alpha_inv, "alpha_inv", torch.float32), float(eps), B, C, T, lay,
              _dev(out, "out", torch.float32), _stream(x))
    return out


# ------------------------------------------------------------- HiFT DSP --

NSF_HARMONICS = 9


def hann_window(n_fft: int = 16) -> np.ndarray:
    """Host periodic Hann window, the engine's f32 expression (hift_vocoder.cpp:429-434)."""
    out = np.empty(n_fft, np.float32)
    _lib.call("cbx_hann_window", int(n_fft), out.ctypes.data_as(ctypes.c_void_p))
    return out


@_on_tensor_device
def nsf_source(f0: torch.Tensor, upsample: int, phase: torch.Tensor, noise: torch.Tensor,
               lin_w, lin_b: float = 0.0, sampling_rate: int = 24000,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """HiFT harmonic source (hift_vocoder.cpp:853-965) with explicit phase and noise.

    f0: f32 [B, n_mel] (or [n_mel]); phase: f32 [B, 9]; noise: f32 [B, 9, n_mel * upsample];
    lin_w: the 9 l_linear weights (host sequence); returns f32 [B, n_mel * upsample]."""
    f2 = f0.unsqueeze(0) if f0.dim() == 1 else f0
    B, n_mel = f2.shape
    T = n_mel * int(upsample)
    if phase.numel() != B * NSF_HARMONICS or noise.numel() != B * NSF_HARMONICS * T:
        raise ValueError("phase must hold B*9 and noise B*9*n_mel*upsample values")
    w = np.ascontiguousarray(np.asarray(lin_w, np.float32).reshape(-1))
    if w.size != NSF_HARMONICS:
        raise ValueError("lin_w must hold 9 weights")
    if out is None:
        out = torch.empty((B, T), dtype=torch.float32, device=f0.device)
    _lib.call("cbx_nsf_source", _dev(f2, "f0", torch.float32), B, n_mel, int(upsample),
              int(sampling_rate), _dev(phase, "phase", torch.float32),
              _dev(noise, "noise", torch.float32), w.ctypes.data_as(ctypes.c_void_p),
              float(lin_b), _dev(out, "out", torch.float32), _stream(f0))
    return out


@_on_tensor_device
def stft(audio: torch.Tensor, n_fft: int = 16, hop: int = 4, window: torch.Tensor | None = None,
         layout="BTC", out: torch.Tensor | None = None) -> torch.Tensor:
    """Centered STFT (hift_vocoder.cpp:465-498) of f32 audio [B, T] (or [T]).

    BTC -> [B, T_stft, 2*nb] (real bins then imag bins per frame); BCT -> [B, 2*nb, T_stft]."""
    lay = _layout(layout)
    a2 = audio.unsqueeze(0) if audio.dim() == 1 else audio
    B, T = a2.shape
    if window is None:
        window = torch.from_numpy(hann_window(n_fft)).to(audio.device)
    nb = n_fft // 2 + 1
    Ts = 1 + T // hop
    if out is None:
        shape = (B, Ts, 2 * nb) if lay == BTC else (B, 2 * nb, Ts)
        out = torch.empty(shape, dtype=torch.float32, device=audio.device)
    _lib.call("cbx_stft", _dev(a2, "audio", torch.float32), B, T, int(n_fft), int(hop),
              _dev(window, "window", torch.float32), lay, _dev(out, "out", torch.float32),
              _stream(audio))
    return out


@_on_tensor_device
def istft_post(post: torch.Tensor, n_fft: int = 16, hop: int = 4,
               window: torch.Tensor | None = None, layout="BTC", audio_limit: float = 0.99,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """HiFT output tail (hift_vocoder.cpp:787-829): conv_post channels -> magnitude / phase ->
    centered iSTFT -> clamp.  post: f32 BTC [B, T_f, 2*nb] or BCT [B, 2*nb, T_f] (2-D: one
    item); returns f32 [B, (T_f - 1) * hop]."""
    lay = _layout(layout)
    p3 = post.unsqueeze(0) if post.dim() == 2 else post
    B = p3.shape[0]
    Tf = p3.shape[1] if lay == BTC else p3.shape[2]
    if window is None:
        window = torch.from_numpy(hann_window(n_fft)).to(post.device)
    if out is None:
        out = torch.empty((B, (Tf - 1) * hop), dtype=torch.float32, device=post.device)
    _lib.call("cbx_istft_post", _dev(p3, "post", torch.float32), B, Tf, int(n_fft), int(hop),
              _dev(window, "window", torch.float32), lay, float(audio_limit),
              _dev(out, "out", torch.float32), _stream(post))
    return out


# ------------------------------------------------------- T3 QKV epilogue --

@_on_tensor_device
def qkv_kv_append(qkv: torch.Tensor, bias: torch.Tensor | None, cache_k: torch.Tensor,
                  cache_v: torch.Tensor, positions: torch.Tensor | None = None,
                  pos_offset: int = 0, slab_stride: int = 0, max_context: int | None = None,
                  err: torch.Tensor | None = None, with_q: bool = True):
    """qkv bias add + Q + KV-cache writes (t3.cpp:465-489).

    qkv: f32 [n_rows, 3D]; bias: f32 [3D] or None; cache_k / cache_v: f32 / f16 / bf16
    buffers addressed as cache[r * slab_stride + pos * D + i]; positions: int32 [n_rows]
    (None: pos_offset + r).  Returns (q [n_rows, D] f32 or None, err int32 [1] device)."""
    if qkv.dim() != 2:
        raise ValueError(f"qkv must be 2-D [n_rows, 3D], got shape {tuple(qkv.shape)}")
    n_rows, D3 = qkv.shape
    if D3 % 3:
        raise ValueError(f"qkv's row length {D3} is not a multiple of 3")
    D = D3 // 3
    if max_context is None:
        raise ValueError("max_context required")
    max_context, slab_stride = int(max_context), int(slab_stride)
    if max_context <= 0 or slab_stride < 0:
        raise ValueError(f"max_context {max_context} / slab_stride {slab_stride}")
    if cache_k.dtype != cache_v.dtype:
        raise TypeError("cache_k and cache_v must share a dtype")
    # The kernel writes cache[r * slab_stride + pos * D + i] for pos in
    # [0, max_context): every such element must lie inside both caches, and
    # per-row slabs must not overlap.
    if n_rows > 1 and slab_stride and slab_stride < max_context * D:
        raise ValueError(f"slab_stride {slab_stride} < max_context * D = {max_context * D}: "
                         "the rows' cache slabs would overlap")
    need = (n_rows - 1) * slab_stride + max_context * D if n_rows else 0
    if cache_k.numel() != cache_v.numel() or cache_k.numel() < need:
        raise ValueError(f"caches hold {cache_k.numel()} / {cache_v.numel()} elements; "
                         f"{n_rows} rows at slab_stride {slab_stride} and max_context "
                         f"{max_context} need {need} in each")
    if positions is not None and positions.numel() < n_rows:
        raise ValueError(f"positions has {positions.numel()} entries for {n_rows} rows")
    if bias is not None and bias.numel() != D3:
        raise ValueError(f"bias has {bias.numel()} entries, expected 3D = {D3}")
    if err is not None and err.numel() < 1:
        raise ValueError("err must hold one int32")
    q = torch.empty((n_rows, D), dtype=torch.float32, device=qkv.device) if with_q else None
    if err is None:
        err = torch.zeros(1, dtype=torch.int32, device=qkv.device)
    _lib.call("cbx_qkv_kv_append", _dev(qkv, "qkv", torch.float32), D3,
              _dev(bias, "bias", torch.float32), n_rows, D,
              _dev(positions, "positions", torch.int32), int(pos_offset),
              _dev(cache_k, "cache_k"), _dev(cache_v, "cache_v"), _cbx_type(cache_k),
              int(slab_stride), int(max_context), _dev(q, "q", torch.float32),
              _dev(err, "err", torch.int32), _stream(qkv))
    return q, err


# ------------------------------------------------------- paged KV cache --
#
# A decode step calls these once per layer, and a call of the smallest sizes is bound by its Python
# operations, not by its kernel.  So the checks are few and cheap while all is well, and the full
# message is made where something is not.

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_I32, _F32 = torch.int32, torch.float32


def _on_device(fn):
    """``_on_tensor_device`` in fewer operations: run with the device of the first parameter's tensor
    current, whichever place its keyword has.  The wrappers compare the other tensors with it."""
    first = next(iter(inspect.signature(fn).parameters))

    @functools.wraps(fn)
    def wrapper(*args, **kw):
        t = args[0] if args else kw.get(first)
        dev = t.get_device() if isinstance(t, torch.Tensor) else -1
        if dev >= 0 and dev != _current_device():
            with torch.cuda.device(dev):
                return fn(*args, **kw)
        return fn(*args, **kw)
    return wrapper


@functools.cache
def _fn(name: str):
    """The library's function, looked up once."""
    return getattr(_lib.load(), name)


def _ok(dev: int, dtype, tensors) -> bool:
    """Every tensor (None aside) is dense, of this type and on CUDA device `dev`."""
    try:
        for t in tensors:
            if t is not None and (t.dtype is not dtype or t.get_device() != dev
                                  or not t.is_contiguous()):
                return False
        return dev >= 0
    except AttributeError:  # not a tensor
        return False


def _refuse(dtype, **tensors):
    """Raises what is wrong with one of the tensors."""
    for name, t in tensors.items():
        _dev(t, name, dtype)
    raise ValueError(f"{', '.join(tensors)}: dense CUDA tensors of one device and of {dtype} expected")


def _refuse_strided(**tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (libcbx_ops has no CPU path)")
        if t.device.index != torch.cuda.current_device():
            raise ValueError(f"{name} is on {t.device}, the call runs on "
                             f"cuda:{torch.cuda.current_device()}: all tensors of a call must "
                             "share its device")


def _type_of(t: torch.Tensor) -> int:
    v = _TORCH_TO_CBX.get(t.dtype)
    return _cbx_type(t) if v is None else v


def _err_word(err: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if err is None:
        return torch.zeros(1, dtype=_I32, device=like.device)
    if err.numel() < 1:
        raise ValueError("err must hold one int32")
    return err


def _paged_cache(cache_k: torch.Tensor, cache_v: torch.Tensor):
    """(n_pages, page_size, n_kv_heads, head_dim, page_stride) of two caches
    [n_pages, page_size, n_kv_heads, head_dim]: the last three dimensions dense, the pages a
    fixed stride apart (so a cache can be one layer of a pool [n_pages, n_layers, 2, ...])."""
    shape = cache_k.shape
    if len(shape) != 4 or cache_v.shape != shape:
        raise ValueError("cache_k and cache_v must be [n_pages, page_size, n_kv_heads, head_dim] "
                         f"of one shape, got {tuple(shape)} and {tuple(cache_v.shape)}")
    if cache_k.dtype is not cache_v.dtype:
        raise TypeError("cache_k and cache_v must share a dtype")
    P, S, Hk, hd = shape
    if P * S * Hk * hd == 0:
        raise ValueError(f"the caches are empty: shape {tuple(shape)}")
    page = S * Hk * hd
    if cache_k.is_contiguous() and cache_v.is_contiguous():
        return P, S, Hk, hd, page
    strides = cache_k.stride()
    # the stride of a dimension of one entry means nothing
    dense = all(n == 1 or s == v == d for n, s, v, d in
                zip((S, Hk, hd), strides[1:], cache_v.stride()[1:], (Hk * hd, hd, 1)))
    page_stride = strides[0] if P > 1 else page
    if not dense or page_stride < page or (P > 1 and cache_v.stride(0) != page_stride):
        raise ValueError("the caches' pages must be dense [page_size, n_kv_heads, head_dim] blocks "
                         f"and equally far apart, got strides {strides} and {cache_v.stride()}")
    return P, S, Hk, hd, page_stride


class PagedPlan(NamedTuple):
    """What ``paged_plan`` returns: the step's rows, then the state after it."""
    slots: torch.Tensor        # [max_rows] cache slot of each row, -1: none
    positions: torch.Tensor    # [max_rows]
    row_reqs: torch.Tensor     # [max_rows] request of each row
    row_lens: torch.Tensor     # [max_rows] keys a row attends to: position + 1
    row_start: torch.Tensor    # [n_reqs + 1] first row of each request
    block_table: torch.Tensor  # [n_reqs, max_blocks]
    n_blocks: torch.Tensor     # [n_reqs]
    free_list: torch.Tensor    # [n_pages]
    n_free: torch.Tensor       # [1]
    err: torch.Tensor          # [1] device error word (EFLAG_NO_PAGE, _PAGE_OOB, _LENGTH)


@_on_device
def paged_plan(seq_lens: torch.Tensor, block_table: torch.Tensor, n_blocks: torch.Tensor,
               free_list: torch.Tensor, n_free: torch.Tensor, page_size: int,
               n_new: torch.Tensor | None = None, max_rows: int | None = None,
               in_place: bool = False, out=None, err: torch.Tensor | None = None) -> PagedPlan:
    """Block tables, slots and positions of one step, on the device (see cbx_paged_plan).

    seq_lens: int32 [n_reqs], the tokens each request holds after the step (0: ended or empty);
    n_new: int32 [n_reqs], how many of them, the last ones, the step writes (None: one for each
    request that is there); max_rows: rows to lay out (None: n_reqs).  State: block_table int32
    [n_reqs, max_blocks], n_blocks int32 [n_reqs], free_list int32 [n_pages], n_free int32 [1].
    With ``in_place`` the state tensors are updated, otherwise new ones are returned; ``out``
    (the first 9 tensors of an earlier plan of the same sizes) gives the buffers."""
    n_reqs, n_pages = seq_lens.numel(), free_list.numel()
    if block_table.dim() != 2 or block_table.shape[0] != n_reqs:
        raise ValueError(f"block_table must be [n_reqs, max_blocks], got {tuple(block_table.shape)} "
                         f"for {n_reqs} requests")
    max_blocks = block_table.shape[1]
    if n_blocks.numel() != n_reqs or n_free.numel() != 1 or \
            (n_new is not None and n_new.numel() != n_reqs):
        raise ValueError("n_blocks and n_new must hold n_reqs entries, n_free one")
    max_rows = n_reqs if max_rows is None else int(max_rows)
    if out is not None:
        if in_place:
            raise ValueError("out and in_place exclude one another")
        out = tuple(out)[:9]
        sizes = [max_rows, max_rows, max_rows, max_rows, n_reqs + 1, n_reqs * max_blocks, n_reqs,
                 n_pages, 1]
        if [t.numel() for t in out] != sizes:
            raise ValueError(f"out must hold 9 tensors of {sizes} entries")
    else:
        def new(n):
            return torch.empty(n, dtype=_I32, device=seq_lens.device)
        rows = [new(max_rows) for _ in range(4)] + [new(n_reqs + 1)]
        state = (block_table, n_blocks, free_list, n_free)
        out = (*rows, *(state if in_place else map(torch.empty_like, state)))
    dev = seq_lens.get_device()
    if not _ok(dev, _I32, (seq_lens, n_new, block_table, n_blocks, free_list, n_free, err, *out)):
        _refuse(_I32, seq_lens=seq_lens, n_new=n_new, block_table=block_table, n_blocks=n_blocks,
                free_list=free_list, n_free=n_free, err=err,
                **{f"out[{i}]": t for i, t in enumerate(out)})
    err = _err_word(err, seq_lens)
    slots, positions, row_reqs, row_lens, row_start, table_o, blocks_o, free_o, n_free_o = [
        t.data_ptr() for t in out]
    status = _fn("cbx_paged_plan")(
        seq_lens.data_ptr(), None if n_new is None else n_new.data_ptr(), n_reqs, max_blocks,
        int(page_size), n_pages, block_table.data_ptr(), n_blocks.data_ptr(), free_list.data_ptr(),
        n_free.data_ptr(), table_o, blocks_o, free_o, n_free_o, max_rows, slots, positions,
        row_reqs, row_lens, row_start, err.data_ptr(), _raw_stream(dev))
    if status:
        _lib.check("cbx_paged_plan", status)
    return PagedPlan(*out, err)


@_on_device
def qkv_kv_append_paged(qkv: torch.Tensor, bias: torch.Tensor | None, cache_k: torch.Tensor,
                        cache_v: torch.Tensor, slots: torch.Tensor,
                        q_out: torch.Tensor | None = None, err: torch.Tensor | None = None,
                        with_q: bool = True):
    """qkv bias add + Q + K / V written into pages (t3.cpp:465-489 on a paged cache).

    qkv: f32 / f16 / bf16 [n_rows, q_dim + 2 kv_dim] (rows may be strided); bias: f32 or None;
    caches [n_pages, page_size, n_kv_heads, head_dim]; slots: int32 [n_rows], page * page_size +
    place, -1 skips the row.  Returns (q [n_rows, q_dim] of qkv's dtype or None, err).  The q
    rows of skipped rows are left as they were in q_out (without q_out: unspecified)."""
    if qkv.dim() != 2:
        raise ValueError(f"qkv must be 2-D [n_rows, q_dim + 2 kv_dim], got shape {tuple(qkv.shape)}")
    n_rows, width = qkv.shape
    stride = width
    if not qkv.is_contiguous():
        if width > 1 and qkv.stride(1) != 1:
            raise ValueError(f"qkv's rows must be dense, got strides {qkv.stride()}")
        stride = qkv.stride(0) if n_rows > 1 else width
        if stride < width:
            raise ValueError(f"qkv's rows overlap: stride {stride} < {width}")
    P, S, Hk, hd, page_stride = _paged_cache(cache_k, cache_v)
    kv_dim = Hk * hd
    q_dim = width - 2 * kv_dim
    if q_dim < 0:
        raise ValueError(f"qkv's row length {width} is below 2 kv_dim = {2 * kv_dim}")
    if slots.numel() < n_rows:
        raise ValueError(f"slots has {slots.numel()} entries for {n_rows} rows")
    if bias is not None and bias.numel() != width:
        raise ValueError(f"bias has {bias.numel()} entries, expected {width}")
    if q_out is not None and q_out.numel() != n_rows * q_dim:
        raise ValueError(f"q_out must hold {n_rows} x {q_dim} values of {qkv.dtype}")
    dev = qkv.get_device()
    if cache_k.get_device() != dev or cache_v.get_device() != dev or dev < 0:
        _refuse_strided(qkv=qkv, cache_k=cache_k, cache_v=cache_v)
    if not _ok(dev, _I32, (slots, err)):
        _refuse(_I32, slots=slots, err=err)
    if bias is not None and not _ok(dev, _F32, (bias,)):
        _refuse(_F32, bias=bias)
    if q_out is None:
        if with_q:
            q_out = torch.empty((n_rows, q_dim), dtype=qkv.dtype, device=qkv.device)
    elif not _ok(dev, qkv.dtype, (q_out,)):
        _refuse(qkv.dtype, q_out=q_out)
    if err is None or err.numel() != 1:
        err = _err_word(err, qkv)
    status = _fn("cbx_qkv_kv_append_paged")(
        qkv.data_ptr(), _type_of(qkv), stride, None if bias is None else bias.data_ptr(), n_rows,
        q_dim, kv_dim, slots.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(), _type_of(cache_k),
        P, S, page_stride, None if q_out is None else q_out.data_ptr(), err.data_ptr(),
        _raw_stream(dev))
    if status:
        _lib.check("cbx_qkv_kv_append_paged", status)
    return q_out, err


@_on_device
def paged_decode_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor,
                           block_table: torch.Tensor, seq_lens: torch.Tensor,
                           row_reqs: torch.Tensor | None = None, scale: float | None = None,
                           return_lse: bool = False, out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None,
                           err: torch.Tensor | None = None):
    """softmax(scale q K^T) V of one new token per row over a paged cache.

    q: [n_rows, n_heads, head_dim] f32 / f16 / bf16 (rows may be strided); caches [n_pages,
    page_size, n_kv_heads, head_dim]; block_table: int32 [n_reqs, max_blocks]; seq_lens: int32
    [n_rows], the keys of each row (0: zeros); row_reqs: int32 [n_rows], each row's request (None:
    row r is request r); scale: head_dim ** -0.5 by default.  Returns out [n_rows, n_heads,
    head_dim] of q's dtype, with ``return_lse`` (out, lse f32 [n_rows, n_heads]).  ``workspace``:
    a byte tensor of ``paged_decode_attention_workspace`` bytes to use instead of a new one."""
    if q.dim() != 3:
        raise ValueError(f"q must be [n_rows, n_heads, head_dim], got shape {tuple(q.shape)}")
    n_rows, H, qd = q.shape
    q_stride = H * qd
    if not q.is_contiguous():
        if q.numel() > 0 and not q[0].is_contiguous():
            raise ValueError(f"q's rows must be dense, got strides {q.stride()}")
        q_stride = q.stride(0) if n_rows > 1 else H * qd
        if q_stride < H * qd:
            raise ValueError(f"q's rows overlap: stride {q_stride}")
    P, S, Hk, hd, page_stride = _paged_cache(cache_k, cache_v)
    if qd != hd:
        raise ValueError(f"q's head_dim {qd} is not the caches' {hd}")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [n_reqs, max_blocks], got {tuple(block_table.shape)}")
    n_reqs, max_blocks = block_table.shape
    if seq_lens.numel() != n_rows or (row_reqs is not None and row_reqs.numel() != n_rows):
        raise ValueError(f"seq_lens and row_reqs must hold one entry for each of {n_rows} rows")
    if row_reqs is None and n_reqs < n_rows:
        raise ValueError(f"block_table has {n_reqs} rows for {n_rows} rows of q")
    if out is not None and out.numel() != n_rows * H * hd:
        raise ValueError(f"out must hold {n_rows} x {H} x {hd} values of {q.dtype}")
    dev = q.get_device()
    if cache_k.get_device() != dev or cache_v.get_device() != dev or dev < 0:
        _refuse_strided(q=q, cache_k=cache_k, cache_v=cache_v)
    if not _ok(dev, _I32, (block_table, seq_lens, row_reqs, err)):
        _refuse(_I32, block_table=block_table, seq_lens=seq_lens, row_reqs=row_reqs, err=err)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif not _ok(dev, q.dtype, (out,)):
        _refuse(q.dtype, out=out)
    lse = torch.empty((n_rows, H), dtype=_F32, device=q.device) if return_lse else None
    ct = _type_of(cache_k)
    need = _workspace_bytes(dev, n_rows, H, Hk, hd, max_blocks, S, ct)
    ws_p, ws_bytes = None, 0
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif not _ok(dev, workspace.dtype, (workspace,)):
            _refuse(workspace.dtype, workspace=workspace)
        ws_p, ws_bytes = workspace.data_ptr(), workspace.nbytes
    if err is None or err.numel() != 1:
        err = _err_word(err, q)
    status = _fn("cbx_paged_decode_attention")(
        q.data_ptr(), _type_of(q), q_stride, cache_k.data_ptr(), cache_v.data_ptr(), ct, P, S,
        page_stride, block_table.data_ptr(), n_reqs, max_blocks,
        None if row_reqs is None else row_reqs.data_ptr(), seq_lens.data_ptr(), n_rows, H, Hk, hd,
        hd ** -0.5 if scale is None else scale, out.data_ptr(),
        None if lse is None else lse.data_ptr(), ws_p, ws_bytes, err.data_ptr(), _raw_stream(dev))
    if status:
        _lib.check("cbx_paged_decode_attention", status)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(dev, n_rows, n_heads, n_kv_heads, head_dim, max_blocks, page_size, cache_type):
    """Per device: the split depends on its number of SMs."""
    n = _lib.load().cbx_paged_decode_attention_workspace(n_rows, n_heads, n_kv_heads, head_dim,
                                                         max_blocks, page_size, cache_type)
    if n < 0:
        _lib.check("cbx_paged_decode_attention_workspace", int(n))
    return n


def paged_decode_attention_workspace(n_rows: int, n_heads: int, n_kv_heads: int, head_dim: int,
                                     max_blocks: int, page_size: int,
                                     cache_dtype: torch.dtype = torch.float32) -> int:
    """Bytes of workspace ``paged_decode_attention`` needs for these sizes on the current device."""
    return _workspace_bytes(torch.cuda.current_device(), int(n_rows), int(n_heads),
                            int(n_kv_heads), int(head_dim), int(max_blocks), int(page_size),
                            _TORCH_TO_CBX[cache_dtype])


# ------------------------------------------------- token log probabilities --

class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns (natural logarithms, f32)."""
    logprobs: torch.Tensor | None      # [n_rows] of the given tokens
    entropy: torch.Tensor              # [n_rows]
    top_ids: torch.Tensor              # [n_rows, top_k] int32
    top_logprobs: torch.Tensor         # [n_rows, top_k]
    err: torch.Tensor                  # [1] device error word (EFLAG_TOKEN_OOB)


@_on_device
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None, top_k: int = 0,
                   err: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probabilities of given tokens, entropy and the top_k most probable alternatives.

    logits: f32 / f16 / bf16 [n_rows, vocab] (rows may be strided); tokens: int32 [n_rows] (-1: no
    token, NaN) or None; ties among the alternatives go to the lowest id."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be 2-D [n_rows, vocab], got shape {tuple(logits.shape)}")
    n_rows, vocab = logits.shape
    stride = vocab
    if not logits.is_contiguous():
        if vocab > 1 and logits.stride(1) != 1:
            raise ValueError(f"logits' rows must be dense, got strides {logits.stride()}")
        stride = logits.stride(0) if n_rows > 1 else vocab
        if stride < vocab:
            raise ValueError(f"logits' rows overlap: stride {stride} < {vocab}")
    if not 0 <= top_k <= vocab or top_k > _lib.LOGPROBS_MAX_TOP:
        raise ValueError(f"top_k {top_k} outside [0, min(vocab, {_lib.LOGPROBS_MAX_TOP})]")
    if tokens is not None and tokens.shape != (n_rows,):
        raise ValueError(f"tokens has shape {tuple(tokens.shape)}, not one entry for each of {n_rows} rows")
    dev = logits.get_device()
    if dev < 0:
        _refuse_strided(logits=logits)
    if not _ok(dev, _I32, (tokens, err)):
        _refuse(_I32, tokens=tokens, err=err)
    if tokens is not None:
        lp = torch.empty_like(tokens, dtype=_F32)
        entropy = torch.empty_like(lp)
    else:
        lp, entropy = None, torch.empty(n_rows, dtype=_F32, device=logits.device)
    top = torch.empty((n_rows, top_k), dtype=_F32, device=logits.device)
    ids = torch.empty_like(top, dtype=_I32)
    if err is None or err.numel() != 1:
        err = _err_word(err, logits)
    status = _fn("cbx_token_logprobs")(
        logits.data_ptr(), _type_of(logits), stride, n_rows, vocab,
        None if lp is None else tokens.data_ptr(), top_k, None if lp is None else lp.data_ptr(),
        entropy.data_ptr(), ids.data_ptr(), top.data_ptr(), err.data_ptr(), _raw_stream(dev))
    if status:
        _lib.check("cbx_token_logprobs", status)
    return TokenLogprobs(lp, entropy, ids, top, err)
