"""Penalties for repeated tokens, biases and grammar masks on a batch's logits (sm_100a)."""

from __future__ import annotations

import torch

from asdsl_b200.kernels.paged import _I32, _TYPES, _call, _check, _not_cuda, _ptr, _vector


def logits_process(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, lens: torch.Tensor | None = None,
                   prompt_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   bias_ptr: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias_values: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Processed logits [n, vocab] (fp32, bf16 or fp16), in this order for id v of request b:

    * v among the first lens[b] entries of tokens[b] (prompt, then output): x / repetition[b] for x > 0,
      else x * repetition[b];
    * v c > 0 times in the output (entries from prompt_lens[b] on): x - frequency[b] * c - presence[b];
    * v in the request's bias list, bias_ids / bias_values [bias_ptr[b]:bias_ptr[b + 1]]: x + value
      (entries that repeat add up in list order);
    * bit v % 32 of the int32 mask[b, v // 32] clear: -inf.

    Arithmetic in fp32, one rounding at the end.  Any part may be left out; ids outside the vocabulary
    are ignored.  out may be `logits` itself.  For inference: the result carries no gradient.
    """
    _not_cuda(logits, "logits")
    dtype, device, f32 = logits.dtype, logits.device, torch.float32
    if dtype not in (f32, torch.bfloat16, torch.float16):
        raise ValueError(f"logits of {dtype} are not supported")
    _check(logits, "logits", dtype, 2, None)
    n, vocab = logits.shape
    if vocab <= 0 or (logits.stride(1) != 1 and vocab > 1):
        raise ValueError("the rows of logits must be consecutive in memory")
    if out is None:
        out = torch.empty((n, vocab), dtype=dtype, device=device)
    else:
        _check(out, "out", dtype, 2, device)
        if out.shape != logits.shape or (out.stride(1) != 1 and vocab > 1):
            raise ValueError("out must have logits' shape and consecutive rows")
    t_len = t_stride = n_bias = m_stride = 0
    if tokens is not None:
        _check(tokens, "tokens", _I32, 2, device)
        t_len, t_stride = tokens.shape[1], tokens.stride(0)
        if tokens.shape[0] != n or (tokens.stride(1) != 1 and t_len > 1):
            raise ValueError(f"tokens must be [{n}, length] with consecutive rows")
        if lens is None:
            raise ValueError("tokens need lens")
        _vector(lens, "lens", n, device)
        if prompt_lens is not None:
            _vector(prompt_lens, "prompt_lens", n, device)
        if repetition is not None:
            _vector(repetition, "repetition", n, device, f32)
        if frequency is not None:
            _vector(frequency, "frequency", n, device, f32)
        if presence is not None:
            _vector(presence, "presence", n, device, f32)
    elif repetition is not None or frequency is not None or presence is not None:
        raise ValueError("penalties need tokens")
    if bias_ptr is not None:
        _vector(bias_ptr, "bias_ptr", n + 1, device)
        if bias_ids is None or bias_values is None:
            raise ValueError("bias_ptr needs bias_ids and bias_values")
        _vector(bias_ids, "bias_ids", -1, device)
        n_bias = bias_ids.numel()
        _vector(bias_values, "bias_values", n_bias, device, f32)
    elif bias_ids is not None or bias_values is not None:
        raise ValueError("bias_ids and bias_values need bias_ptr")
    if mask is not None:
        _check(mask, "mask", _I32, 2, device)
        if mask.shape[0] != n or mask.shape[1] < (vocab + 31) // 32:
            raise ValueError(f"mask must be [{n}, {(vocab + 31) // 32}]")
        m_stride = mask.stride(0)
        if mask.stride(1) != 1 and mask.shape[1] > 1:
            raise ValueError("the rows of mask must be consecutive in memory")
    _call(device, "asdsl_b200_logits_process", logits.data_ptr(), out.data_ptr(), _TYPES[dtype],
          logits.stride(0), out.stride(0), n, vocab, _ptr(tokens), t_stride, t_len, _ptr(lens), _ptr(prompt_lens),
          _ptr(repetition), _ptr(frequency), _ptr(presence), _ptr(bias_ptr), _ptr(bias_ids), _ptr(bias_values), n_bias,
          _ptr(mask), m_stride)
    return out
