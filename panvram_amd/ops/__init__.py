"""Operators of a recurrent language model over a cohort's windows, as HIP kernels on tensors that are on the GPU.

    gated_scan(gate, value, state, reset)            h[t] = (1 - sigmoid(gate[t])) h[t-1] + sigmoid(gate[t]) value[t]
    gated_delta(query, key, value, gate, write)      a matrix as each head's state, written by the delta rule and read by queries
    add_rms_norm(x, residual, weight)                the residual stream's addition and its root-mean-square norm
    add_rms_norm_8bit(x, residual, weight)           the same with the norm in 8 bits and a scale per row
    add_layer_norm(x, residual, weight, bias)        the addition, with dropout of x, and its layer norm
    dropout(x, p, seed, site)                        elements dropped by a counter-based generator, without a stored mask
    next_base_loss(hidden, weight, tokens)           head and cross-entropy of the next token, over a small alphabet
    next_base_loss_grad(hidden, weight, tokens)      the loss and its gradients in one pass
    gradient_norm(grads), clip_gradients(grads, m)   the norm over many tensors, and the tensors scaled to at most m

gated_scan, gated_delta, add_rms_norm, add_layer_norm, dropout and next_base_loss take part in autograd, backwards;
forward-mode derivatives are refused. Every call runs on the current stream of its tensors' device, waits for nothing, and may
be captured into a graph; what it returns and the scratch memory it uses come from torch's allocator. Types: float32, bfloat16,
float16; sums, norms and states are kept in 32 bits or more. The reference has no counterpart (its
examples/train_small.py trains a stock torch model on the same windows)."""
from .clip import clip_gradients, gradient_norm
from .delta import gated_delta
from .dropout import dropout
from .layer import add_layer_norm
from .loss import next_base_loss, next_base_loss_grad
from .norm import add_rms_norm, add_rms_norm_8bit
from .scan import gated_scan

__all__ = ["gated_scan", "gated_delta", "add_rms_norm", "add_rms_norm_8bit", "add_layer_norm", "dropout", "next_base_loss", "next_base_loss_grad", "gradient_norm",
           "clip_gradients"]
