"""Operators on sequences of tokens (include/aclnn_sequence.h) over torch CUDA tensors: one native call each, on the current stream of
the tensors' device. Results are allocated unless they are given; a workspace is used by one call at a time."""
import torch

from .aclnn import native

__all__ = [
    "residual_rms_norm", "residual_rms_norm_backward", "residual_rms_norm_quant", "rotary_embedding", "rotary_embedding_backward",
    "rotary_frequencies", "window_attention", "window_attention_backward",
]


def residual_rms_norm(x, residual=None, weight=None, eps=1e-6, out=None, sum_out=None, rstd_out=None, workspace=None):
    """(y, sum, rstd): sum = x + residual in x's type (x itself without a residual), y = sum * rstd * weight with
    rstd = 1 / sqrt(mean(sum^2) + eps) over the last dimension, in fp32."""
    return native().residual_rms_norm(x, residual, weight, eps, out, sum_out, rstd_out, workspace)


def residual_rms_norm_backward(grad_y, sum, rstd, weight=None, grad_sum=None, grad_x=None, grad_weight=None, workspace=None):
    """(grad_x, grad_weight) from the sum and rstd that the forward returned; grad_x is the gradient of x and of residual.
    grad_sum: the gradient that reaches the sum by its other use. grad_weight is None without a weight."""
    return native().residual_rms_norm_backward(grad_y, sum, rstd, weight, grad_sum, grad_x, grad_weight, workspace)


def residual_rms_norm_quant(x, residual=None, weight=None, eps=1e-6, dtype=torch.float8_e4m3fn, group=0, out=None, scales_out=None,
                            sum_out=None, workspace=None):
    """(q, scales, sum): the norm in 8 bits (torch.float8_e4m3fn or torch.int8), y being about q * scale, with one scale a row
    (group 0) or one for each `group` columns."""
    if dtype not in (torch.float8_e4m3fn, torch.int8):
        raise ValueError(f"dtype must be torch.float8_e4m3fn or torch.int8, got {dtype}")
    return native().residual_rms_norm_quant(x, residual, weight, eps, dtype == torch.int8, group, out, scales_out, sum_out, workspace)


def rotary_embedding(q, k, positions, frequencies, interleaved=False, sections=None, scale=1.0, q_out=None, k_out=None,
                     workspace=None):
    """(q', k') with the first 2 * len(frequencies) values of each head turned by position * frequency; k may be None.
    q is [..., heads, dim]; positions has (or broadcasts to) its leading dimensions, behind a dimension of the axes where `sections`
    are given: [axes, tokens] serves all sequences of q [batch, tokens, heads, dim]. Pairs are (i, half + i), or neighbours where `interleaved`. q_out may be q and k_out k."""
    return native().rotary_embedding(q, k, positions, frequencies, interleaved, sections, scale, q_out, k_out, workspace, False)


def rotary_embedding_backward(grad_q_out, grad_k_out, positions, frequencies, interleaved=False, sections=None, scale=1.0, grad_q=None,
                              grad_k=None, workspace=None):
    """(grad_q, grad_k): the turn by the negative angles; the arguments are those of the forward."""
    return native().rotary_embedding(grad_q_out, grad_k_out, positions, frequencies, interleaved, sections, scale, grad_q, grad_k,
                                     workspace, True)


_SCALINGS = {None: 0, "linear": 1, "base": 2, "wavelength": 3, "ramp": 4}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=0.0, low=1.0, high=4.0,
                       dtype=torch.float32, device="cuda", out=None):
    """The rotary_dim / 2 frequencies base^(-2i / rotary_dim), scaled for contexts `factor` times the trained length: "linear",
    "base", "wavelength" or "ramp" (include/aclnn_sequence.h says how)."""
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of {list(_SCALINGS)}, got {scaling!r}")
    if out is None:
        if rotary_dim < 0 or rotary_dim % 2 != 0:
            raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
        out = torch.empty(rotary_dim // 2, dtype=dtype, device=device)
    return native().rotary_frequencies(out, base, _SCALINGS[scaling], factor, original_length, low, high)


def window_attention(q, k, v, window, sinks=0, scale=None, q_lengths=None, kv_lengths=None, out=None, lse=None, workspace=None):
    """(out, lse) of causal attention over the last `window` keys and the first `sinks`: q [batch, queries, heads, dim] against k and
    v [batch, keys, kv heads, dim]; scale is 1 / sqrt(dim) unless given. Sequence b has q_lengths[b] queries and kv_lengths[b] keys
    (all of them unless given), its last query at its last key. lse [batch, heads, queries] is what the backward needs."""
    return native().window_attention(q, k, v, q_lengths, kv_lengths, window, sinks, scale, out, lse, workspace)


def window_attention_backward(grad_out, q, k, v, out, lse, window, sinks=0, scale=None, q_lengths=None, kv_lengths=None, grad_q=None,
                              grad_k=None, grad_v=None, workspace=None):
    """(grad_q, grad_k, grad_v) from the forward's out and lse; the other arguments are the forward's."""
    return native().window_attention_backward(grad_out, q, k, v, out, lse, q_lengths, kv_lengths, window, sinks, scale, grad_q, grad_k,
                                              grad_v, workspace)
