"""trs_views over PyTorch CUDA tensors, and thin callers of the C ABI that
allocate their outputs with PyTorch.

PyTorch only provides device memory and the current stream here; every
computation is a libtrs_b200.so kernel.  Views are described over a tensor's
underlying storage, so any strides the reference can express (including the
negative strides of step_slice, which PyTorch views cannot hold) are passed as
explicit (shape, strides, offset) triples.
"""
from __future__ import annotations

import ctypes

import torch

from . import abi

TORCH_TO_TRS = {torch.float32: abi.F32, torch.float64: abi.F64, torch.int32: abi.I32, torch.int64: abi.I64}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: int | None = None) -> int:
    """PyTorch's current stream of the current device (`device`, where the caller has asked for it already; read straight
    from the binding where it offers that: the Stream object costs 3 us, as much as a launch)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device() if device is None else device)
    return torch.cuda.current_stream().cuda_stream


_DTYPES = {t: (code, abi.DTYPE_SIZE[code]) for t, code in TORCH_TO_TRS.items()}


def view_of(t: torch.Tensor, shape=None, strides=None, offset=None) -> abi.View:
    """A trs_view into t's storage.  Without overrides it describes t itself."""
    if not t.is_cuda:
        raise ValueError("view_of needs a CUDA tensor")
    st = t.untyped_storage()
    code, size = _DTYPES[t.dtype]
    if shape is None and strides is None and offset is None:
        v = abi.pack_view(st.data_ptr(), st.nbytes() // size, code, t.shape, t.stride(), t.storage_offset())
        v.device = t.get_device()
        return v
    if shape is None or list(shape) == list(t.shape):
        shape = t.shape
        if strides is None:
            strides = t.stride()
    if offset is None:
        offset = t.storage_offset()
    v = abi.make_view(st.data_ptr(), code, shape, strides, offset, st.nbytes() // size)
    v.device = t.get_device()
    return v


def _call(name: str, *args) -> int:
    lib = abi.load()
    return abi.check(getattr(lib, name)(*args))


def binary(op: str, a: abi.View, b: abi.View, out: torch.Tensor) -> torch.Tensor:
    _call("trs_binary", abi.BINOPS[op], ctypes.byref(a), ctypes.byref(b), ctypes.byref(view_of(out)),
          stream_handle())
    return out


def unary(op: str, x: abi.View, out: torch.Tensor, p0=0.0, p1=0.0) -> torch.Tensor:
    params = (abi.Scalar * 2)(abi.scalar(p0), abi.scalar(p1))
    _call("trs_unary", abi.UNOPS[op], ctypes.byref(x), params, ctypes.byref(view_of(out)), stream_handle())
    return out


def elementwise(prog: abi.Program, ins: list[abi.View], out: torch.Tensor | None,
                sum_out: torch.Tensor | None = None) -> None:
    arr = abi.views_array(ins)
    ov = ctypes.byref(view_of(out)) if out is not None else None
    if sum_out is None:
        _call("trs_elementwise", ctypes.byref(prog), arr, ov, stream_handle())
    else:
        _call("trs_elementwise_sum", ctypes.byref(prog), arr, ov, ctypes.byref(view_of(sum_out)),
              stream_handle())


def elementwise_row_sums(prog: abi.Program, ins: list[abi.View], out: torch.Tensor,
                         row_sums: torch.Tensor | None, total: torch.Tensor | None) -> None:
    """Y = prog(ins) into `out`, its sums along the last axis into `row_sums`
    and its total into `total`, in one pass (trs_elementwise_row_sums)."""
    arr = abi.views_array(ins)
    rv = ctypes.byref(view_of(row_sums)) if row_sums is not None else None
    tv = ctypes.byref(view_of(total)) if total is not None else None
    _call("trs_elementwise_row_sums", ctypes.byref(prog), arr, ctypes.byref(view_of(out)), rv, tv,
          stream_handle())


def pack(x: abi.View, out: torch.Tensor) -> torch.Tensor:
    _call("trs_pack", ctypes.byref(x), ctypes.byref(view_of(out)), stream_handle())
    return out


def sum_all(x: abi.View, out: torch.Tensor) -> torch.Tensor:
    _call("trs_sum", ctypes.byref(x), ctypes.byref(view_of(out)), stream_handle())
    return out


def sum_axis(x: abi.View, axis: int, keepdim: bool, out: torch.Tensor) -> torch.Tensor:
    _call("trs_sum_axis", ctypes.byref(x), axis, int(keepdim), ctypes.byref(view_of(out)), stream_handle())
    return out


def mean_axis(x: abi.View, axis: int, keepdim: bool, out: torch.Tensor) -> torch.Tensor:
    _call("trs_mean_axis", ctypes.byref(x), axis, int(keepdim), ctypes.byref(view_of(out)), stream_handle())
    return out


def max_axis(x: abi.View, axis: int, out: torch.Tensor) -> torch.Tensor:
    _call("trs_max_axis", ctypes.byref(x), axis, ctypes.byref(view_of(out)), stream_handle())
    return out


def argmax_axis(x: abi.View, axis: int, out: torch.Tensor) -> torch.Tensor:
    _call("trs_argmax_axis", ctypes.byref(x), axis, ctypes.byref(view_of(out)), stream_handle())
    return out


def reduce_broadcast_grad(g: abi.View, target: list[int], out: torch.Tensor) -> int:
    """Returns abi.OK, or abi.NONE where the reference returns None."""
    t = (ctypes.c_int64 * max(1, len(target)))(*target)
    return _call("trs_reduce_broadcast_grad", ctypes.byref(g), t, len(target), ctypes.byref(view_of(out)),
                 stream_handle())


def sum_to_shape_fused(g: abi.View, gate: abi.View | None, mul: abi.View | None, target: list[int],
                       out: torch.Tensor) -> int:
    t = (ctypes.c_int64 * max(1, len(target)))(*target)
    return _call("trs_sum_to_shape_fused", ctypes.byref(g), ctypes.byref(gate) if gate is not None else None,
                 ctypes.byref(mul) if mul is not None else None, t, len(target), ctypes.byref(view_of(out)),
                 stream_handle())


def affine_relu_backward(g: abi.View, x: abi.View, scale: abi.View, bias: abi.View,
                         grad_scale: torch.Tensor | None, grad_bias: torch.Tensor | None) -> None:
    _call("trs_affine_relu_backward", ctypes.byref(g), ctypes.byref(x), ctypes.byref(scale), ctypes.byref(bias),
          ctypes.byref(view_of(grad_scale)) if grad_scale is not None else None,
          ctypes.byref(view_of(grad_bias)) if grad_bias is not None else None, stream_handle())


def softmax_lastdim(x: abi.View, out: torch.Tensor) -> torch.Tensor:
    _call("trs_softmax_lastdim", ctypes.byref(x), ctypes.byref(view_of(out)), stream_handle())
    return out


def layer_norm_lastdim(x: abi.View, gamma: abi.View, beta: abi.View, eps: float, out: torch.Tensor) -> torch.Tensor:
    """LayerNorm::forward over the last axis (nn/layer_norm.rs:20-33)."""
    _call("trs_layer_norm_lastdim", ctypes.byref(x), ctypes.byref(gamma), ctypes.byref(beta), float(eps),
          ctypes.byref(view_of(out)), stream_handle())
    return out


def sgd_step(param: torch.Tensor, grad: torch.Tensor, lr: float) -> None:
    """SGD::step for one parameter (optim/sgd.rs:29-37), in place."""
    _call("trs_sgd_step", ctypes.byref(view_of(param)), ctypes.byref(view_of(grad)), float(lr), stream_handle())


def rmsprop_step(param: torch.Tensor, grad: torch.Tensor, v: torch.Tensor, lr: float, alpha: float = 0.99,
                 eps: float = 1e-8) -> None:
    """RMSprop::step for one parameter (optim/rmsprop.rs:30-46), in place."""
    _call("trs_rmsprop_step", ctypes.byref(view_of(param)), ctypes.byref(view_of(grad)), ctypes.byref(view_of(v)),
          float(lr), float(alpha), float(eps), stream_handle())


def adam_step(param: torch.Tensor, grad: torch.Tensor, m: torch.Tensor, v: torch.Tensor, lr: float, t: int,
              beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8) -> None:
    """Adam::step for one parameter at step t >= 1 (optim/adam.rs:119-144), in place."""
    _call("trs_adam_step", ctypes.byref(view_of(param)), ctypes.byref(view_of(grad)), ctypes.byref(view_of(m)),
          ctypes.byref(view_of(v)), float(lr), float(beta1), float(beta2), float(eps), int(t), stream_handle())


def pooled_size(size: tuple[int, int], kernel: tuple[int, int], stride: tuple[int, int]) -> tuple[int, int]:
    """The spatial size a pooling layer turns `size` into (pooled_size, nn/pool.rs:8-17;
    MaxPool2d::output_size / AvgPool2d::output_size).  No padding: a window that
    would hang over the edge is not taken."""
    if stride[0] <= 0 or stride[1] <= 0:
        raise ValueError("!!!MaxPool2d: stride must be positive!!!")
    if size[0] < kernel[0] or size[1] < kernel[1]:
        raise ValueError("the input is smaller than one window")
    return (size[0] - kernel[0]) // stride[0] + 1, (size[1] - kernel[1]) // stride[1] + 1


def max_pool2d(x: abi.View, kernel: tuple[int, int], out: torch.Tensor,
               stride: tuple[int, int] | None = None) -> torch.Tensor:
    """MaxPool2d::forward (nn/pool.rs:137-144) of an [N, C, H, W] view; the stride
    defaults to the kernel (MaxPool2d::new)."""
    sh, sw = stride if stride is not None else kernel
    _call("trs_max_pool2d", ctypes.byref(x), int(kernel[0]), int(kernel[1]), int(sh), int(sw),
          ctypes.byref(view_of(out)), stream_handle())
    return out


def avg_pool2d(x: abi.View, kernel: tuple[int, int], out: torch.Tensor,
               stride: tuple[int, int] | None = None) -> torch.Tensor:
    """AvgPool2d::forward (nn/pool.rs:223-233)."""
    sh, sw = stride if stride is not None else kernel
    _call("trs_avg_pool2d", ctypes.byref(x), int(kernel[0]), int(kernel[1]), int(sh), int(sw),
          ctypes.byref(view_of(out)), stream_handle())
    return out


def max_pool2d_backward(x: abi.View, grad_out: abi.View, kernel: tuple[int, int], grad_x: torch.Tensor,
                        stride: tuple[int, int] | None = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient MaxPool2d passes back to x (max_axis backward, then fold_2d);
    with accumulate, added to what grad_x holds."""
    sh, sw = stride if stride is not None else kernel
    _call("trs_max_pool2d_backward", ctypes.byref(x), ctypes.byref(grad_out), int(kernel[0]), int(kernel[1]),
          int(sh), int(sw), int(bool(accumulate)), ctypes.byref(view_of(grad_x)), stream_handle())
    return grad_x


def matmul_shape(a: abi.View, b: abi.View) -> list[int]:
    """The shape Tensor::matmul returns for a [..., M, K] and b [..., K, N]."""
    sa = [a.shape[i] for i in range(a.ndim)]
    sb = [b.shape[i] for i in range(b.ndim)]
    batch = [max(x, y) for x, y in zip([1] * (len(sb) - len(sa)) + sa[:-2], [1] * (len(sa) - len(sb)) + sb[:-2])]
    return batch + [sa[-2], sb[-1]]


def matmul(a: abi.View, b: abi.View, out: torch.Tensor) -> torch.Tensor:
    """Tensor::matmul (linalg/tensor/base.rs:896-1013), bit-identical to the reference."""
    _call("trs_matmul", ctypes.byref(a), ctypes.byref(b), ctypes.byref(view_of(out)), stream_handle())
    return out


def matmul_tf32x3(a: abi.View, b: abi.View, out: torch.Tensor) -> torch.Tensor:
    """Tensor::matmul for f32 on the tensor cores (split-TF32, within the sum tolerance)."""
    _call("trs_matmul_tf32x3", ctypes.byref(a), ctypes.byref(b), ctypes.byref(view_of(out)), stream_handle())
    return out


def unfold_2d(x: abi.View, kernel, stride, padding, out: torch.Tensor) -> torch.Tensor:
    """Tensor::unfold_2d (linalg/tensor/conv.rs:360-418) into out [B*OH*OW, C*kh*kw]."""
    (kh, kw), (sh, sw), (ph, pw) = kernel, stride, padding
    _call("trs_unfold_2d", ctypes.byref(x), kh, kw, sh, sw, ph, pw, ctypes.byref(view_of(out)), stream_handle())
    return out


def fold_2d(cols: abi.View, kernel, stride, padding, out: torch.Tensor) -> torch.Tensor:
    """Tensor::fold_2d (linalg/tensor/conv.rs:434-488) into out [B, C, H, W]."""
    (kh, kw), (sh, sw), (ph, pw) = kernel, stride, padding
    _call("trs_fold_2d", ctypes.byref(cols), kh, kw, sh, sw, ph, pw, ctypes.byref(view_of(out)), stream_handle())
    return out


# Operands of the attention layer and of a model's ends: inputs are views, outputs tensors, all on the current device.


def _in(v: abi.View | None, here: int):
    if v is None:
        return None
    if v.device != here and v.device is not None:
        raise ValueError("an input lies on another device than the current one")
    return ctypes.byref(v)


def _out(t: torch.Tensor | None, here: int):
    if t is None:
        return None
    if t.get_device() != here:
        raise ValueError("the output lies on another device than the current one")
    return ctypes.byref(view_of(t))


def rotary_frequencies(out: torch.Tensor, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       low_turns: float = 1.0, high_turns: float = 32.0, trained_context: float = 0.0) -> torch.Tensor:
    """The frequencies of rotary positions into out (f64, one per rotated pair);
    scaling as trs_rotary_scaling: none, linear, base, bands or ramp."""
    h = torch.cuda.current_device()
    _call("trs_rotary_frequencies", float(base), abi.ROTARY_SCALINGS[scaling], float(factor), float(low_turns),
          float(high_turns), float(trained_context), _out(out, h), stream_handle(h))
    return out


def rotary(q: abi.View, k: abi.View | None, positions: abi.View, freqs: abi.View, q_out: torch.Tensor,
           k_out: torch.Tensor | None, layout: str = "half", magnitude: float = 1.0) -> None:
    """Rotary positions of q [B, T, Hq, D] and k [B, T, Hk, D]."""
    h = torch.cuda.current_device()
    _call("trs_rotary", _in(q, h), _in(k, h), _in(positions, h), _in(freqs, h), abi.ROTARY_LAYOUTS[layout],
          float(magnitude), _out(q_out, h), _out(k_out, h), stream_handle(h))


def rotary_backward(grad_q_out: abi.View, grad_k_out: abi.View | None, positions: abi.View, freqs: abi.View,
                    grad_q: torch.Tensor, grad_k: torch.Tensor | None, layout: str = "half",
                    magnitude: float = 1.0) -> None:
    """The gradient that rotary passes back to q and k."""
    h = torch.cuda.current_device()
    _call("trs_rotary_backward", _in(grad_q_out, h), _in(grad_k_out, h), _in(positions, h), _in(freqs, h),
          abi.ROTARY_LAYOUTS[layout], float(magnitude), _out(grad_q, h), _out(grad_k, h), stream_handle(h))


def head_norm_rotary(q: abi.View, k: abi.View | None, q_gamma: abi.View | None, k_gamma: abi.View | None, eps: float,
                     positions: abi.View, freqs: abi.View, q_out: torch.Tensor, k_out: torch.Tensor | None,
                     layout: str = "half", magnitude: float = 1.0) -> None:
    """The norm of every head of q and k and its rotation, in one pass."""
    h = torch.cuda.current_device()
    _call("trs_head_norm_rotary", _in(q, h), _in(k, h), _in(q_gamma, h), _in(k_gamma, h), float(eps), _in(positions, h),
          _in(freqs, h), abi.ROTARY_LAYOUTS[layout], float(magnitude), _out(q_out, h), _out(k_out, h), stream_handle(h))


def head_norm_rotary_backward(grad_q_out: abi.View, grad_k_out: abi.View | None, q: abi.View, k: abi.View | None,
                              q_gamma: abi.View | None, k_gamma: abi.View | None, eps: float, positions: abi.View,
                              freqs: abi.View, grad_q: torch.Tensor, grad_k: torch.Tensor | None,
                              grad_q_gamma: torch.Tensor | None, grad_k_gamma: torch.Tensor | None,
                              layout: str = "half", magnitude: float = 1.0) -> None:
    """The gradients of head_norm_rotary for q, k and the gammas."""
    h = torch.cuda.current_device()
    _call("trs_head_norm_rotary_backward", _in(grad_q_out, h), _in(grad_k_out, h), _in(q, h), _in(k, h),
          _in(q_gamma, h), _in(k_gamma, h), float(eps), _in(positions, h), _in(freqs, h), abi.ROTARY_LAYOUTS[layout],
          float(magnitude), _out(grad_q, h), _out(grad_k, h), _out(grad_q_gamma, h), _out(grad_k_gamma, h),
          stream_handle(h))


def cross_attention(q: abi.View, k: abi.View, v: abi.View, scale: float, out: torch.Tensor,
                    lse: torch.Tensor | None = None, key_lengths: abi.View | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v per head: q [B, Tq, Hq, D], k and v [B, Tk, Hk, D], keys of batch b up to
    key_lengths[b]; lse [B, Hq, Tq] is what the backward needs."""
    h = torch.cuda.current_device()
    _call("trs_cross_attention", _in(q, h), _in(k, h), _in(v, h), _in(key_lengths, h), float(scale), _out(out, h),
          _out(lse, h), stream_handle(h))
    return out


def cross_attention_backward(grad_out: abi.View, q: abi.View, k: abi.View, v: abi.View, out: abi.View, lse: abi.View,
                             scale: float, grad_q: torch.Tensor, grad_k: torch.Tensor, grad_v: torch.Tensor,
                             key_lengths: abi.View | None = None) -> None:
    """The gradients of cross_attention for q, k and v."""
    h = torch.cuda.current_device()
    _call("trs_cross_attention_backward", _in(grad_out, h), _in(q, h), _in(k, h), _in(v, h), _in(key_lengths, h),
          _in(out, h), _in(lse, h), float(scale), _out(grad_q, h), _out(grad_k, h), _out(grad_v, h), stream_handle(h))


def embedding(table: abi.View, ids: abi.View, scale: float, out: torch.Tensor) -> torch.Tensor:
    """scale times the rows of table [V, D] that ids name (zeros for ids outside it)."""
    h = torch.cuda.current_device()
    _call("trs_embedding", _in(table, h), _in(ids, h), float(scale), _out(out, h), stream_handle(h))
    return out


def embedding_backward(grad_out: abi.View, ids: abi.View, scale: float, grad_table: torch.Tensor,
                       accumulate: bool = False) -> torch.Tensor:
    """The gradient that embedding passes back to its table; with accumulate, added to what grad_table holds."""
    h = torch.cuda.current_device()
    _call("trs_embedding_backward", _in(grad_out, h), _in(ids, h), float(scale), int(bool(accumulate)),
          _out(grad_table, h), stream_handle(h))
    return grad_table


def linear_cross_entropy(hidden: abi.View, weight: abi.View, targets: abi.View, loss: torch.Tensor,
                         lse: torch.Tensor | None = None, smoothing: float = 0.0) -> torch.Tensor:
    """Softmax cross entropy of hidden weight^T per token, without the logits; lse is what the backward needs."""
    h = torch.cuda.current_device()
    _call("trs_linear_cross_entropy", _in(hidden, h), _in(weight, h), _in(targets, h), float(smoothing), _out(loss, h),
          _out(lse, h), stream_handle(h))
    return loss


def linear_cross_entropy_backward(grad_loss: abi.View, hidden: abi.View, weight: abi.View, targets: abi.View,
                                  lse: abi.View, grad_hidden: torch.Tensor | None, grad_weight: torch.Tensor | None,
                                  smoothing: float = 0.0) -> None:
    """The gradients of linear_cross_entropy for hidden and the weight."""
    h = torch.cuda.current_device()
    _call("trs_linear_cross_entropy_backward", _in(grad_loss, h), _in(hidden, h), _in(weight, h), _in(targets, h),
          _in(lse, h), float(smoothing), _out(grad_hidden, h), _out(grad_weight, h), stream_handle(h))


def linear_distillation(hidden: abi.View, weight: abi.View, teacher_ids: abi.View, teacher_logits: abi.View,
                        temperature: float, loss: torch.Tensor, lse: torch.Tensor | None = None) -> torch.Tensor:
    """The divergence of softmax(hidden weight^T / temperature) from a teacher's largest logits, per token."""
    h = torch.cuda.current_device()
    _call("trs_linear_distillation", _in(hidden, h), _in(weight, h), _in(teacher_ids, h), _in(teacher_logits, h),
          float(temperature), _out(loss, h), _out(lse, h), stream_handle(h))
    return loss


def linear_distillation_backward(grad_loss: abi.View, hidden: abi.View, weight: abi.View, teacher_ids: abi.View,
                                 teacher_logits: abi.View, lse: abi.View, temperature: float,
                                 grad_hidden: torch.Tensor | None, grad_weight: torch.Tensor | None) -> None:
    """The gradients of linear_distillation for hidden and the weight."""
    h = torch.cuda.current_device()
    _call("trs_linear_distillation_backward", _in(grad_loss, h), _in(hidden, h), _in(weight, h), _in(teacher_ids, h),
          _in(teacher_logits, h), _in(lse, h), float(temperature), _out(grad_hidden, h), _out(grad_weight, h),
          stream_handle(h))


def fill_uniform(out: torch.Tensor, seed: int, lo: float = -1.0, hi: float = 1.0, first: int = 0) -> torch.Tensor:
    _call("trs_fill_uniform", ctypes.byref(view_of(out)), seed, first, lo, hi, stream_handle())
    return out


def fill_normal(out: torch.Tensor, seed: int, first: int = 0) -> torch.Tensor:
    _call("trs_fill_normal", ctypes.byref(view_of(out)), seed, first, stream_handle())
    return out
