"""PyTorch operators over the C ABI (the packaging the reference names as its next step, README.md:177).

    import sffft_b200.torch_ops  # registers the operators
    Kf = torch.ops.sffft.filter_spectrum(k)            # k [H][L] fp32 or bf16 -> Kf [H][2L][2] fp32
    y = torch.ops.sffft.conv(u, Kf)                    # u [B][H][L] fp32 or bf16 -> y, same shape and type
    y = sffft_b200.torch_ops.causal_conv(u, k)         # both steps
    y = sffft_b200.torch_ops.two_sided_conv(u, k2)     # non-causal: k2 [H][2L-1], k2[:, L-1] is lag 0
    y = sffft_b200.torch_ops.circular_conv(u, kc)      # period-L circular: kc [H][L]
    X = torch.ops.sffft.rfft(x)                        # x [..., N] fp32/bf16 -> X [..., N/2+1] complex64
    x = torch.ops.sffft.irfft(X)                       # X [..., N/2+1] complex64 -> x [..., N] fp32

    y, S = sffft_b200.torch_ops.linear_attention(q, k, v, log_decay)      # prompts and training, with gradients
    y = sffft_b200.torch_ops.linear_attention_step(q, k, v, log_decay, S) # single tokens, S updated in place
    h, n = sffft_b200.torch_ops.block_norm(x, y, gate, post_weight, weight)   # norms, gate, residual; with gradients

All run on the current CUDA stream of the tensors' device through the C ABI, so they order with surrounding
PyTorch work and can be captured in CUDA graphs (the convolution once a first call has created the plan: plan
creation allocates).  Fake implementations give output shapes and types without running anything, so the operators
trace under torch.compile.  The convolution and the FFTs are forward only (the path has no backward kernel);
linear_attention and block_norm have first derivatives.

`acc` is "fp32" or "fp16" (accumulation mode); `config` names a catalog plan ("" = the default for L).
filter_spectrum and conv must use the same config: the spectrum is in that plan's digit order.
`layout` ("causal", "two_sided", "circular") says which convolution the spectrum makes conv compute; the
fused kernel is the same for all three.
"""
import threading
from typing import Optional

import torch
from torch import Tensor

import sffft_b200 as sf

_plans: dict = {}
_lock = threading.Lock()


def _plan(L: int, io: str, acc: str, config: str, device: int) -> "sf.Plan":
    key = (L, io, acc, config, device)
    with _lock:
        p = _plans.get(key)
        if p is None:
            p = sf.Plan(L, io=io, acc=acc, config=config or None, device=device)
            _plans[key] = p
    return p


def _check_cuda(t: Tensor, what: str):
    if t.device.type != "cuda":
        raise ValueError(f"sffft::{what} needs CUDA tensors (there is no CPU path)")


def _filter_length(k: Tensor, layout: str) -> int:
    """The sequence length L a filter row of this layout belongs to."""
    if layout not in sf.FILTER:
        raise ValueError(f"layout must be one of {sorted(sf.FILTER)}")
    if k.dim() != 2 or k.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("k must be a 2-D float32 or bfloat16 tensor")
    width = k.shape[1]
    if layout == "two_sided":
        if width % 2 == 0:
            raise ValueError("a two-sided filter has 2L-1 taps")
        return (width + 1) // 2
    return width


@torch.library.custom_op("sffft::filter_spectrum", mutates_args=())
def filter_spectrum(k: Tensor, config: str = "", layout: str = "causal") -> Tensor:
    _check_cuda(k, "filter_spectrum")
    L = _filter_length(k, layout)
    H = k.shape[0]
    dev = k.device.index if k.device.index is not None else torch.cuda.current_device()
    plan = _plan(L, "fp32", "fp32", config, dev)
    Kf = torch.empty((H, 2 * L, 2), dtype=torch.float32, device=k.device)
    return plan.filter_spectrum(k.contiguous(), Kf, stream=torch.cuda.current_stream(k.device), layout=layout)


@filter_spectrum.register_fake
def _(k: Tensor, config: str = "", layout: str = "causal") -> Tensor:
    L = _filter_length(k, layout)
    return k.new_empty((k.shape[0], 2 * L, 2), dtype=torch.float32)


@torch.library.custom_op("sffft::conv", mutates_args=())
def conv(u: Tensor, Kf: Tensor, acc: str = "fp32", config: str = "") -> Tensor:
    _check_cuda(u, "conv")
    if u.dim() != 3 or u.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("u must be [B][H][L], float32 or bfloat16")
    B, H, L = u.shape
    if tuple(Kf.shape) != (H, 2 * L, 2) or Kf.dtype != torch.float32 or Kf.device != u.device:
        raise ValueError("Kf must be the [H][2L][2] float32 spectrum on u's device")
    io = "bf16" if u.dtype == torch.bfloat16 else "fp32"
    dev = u.device.index if u.device.index is not None else torch.cuda.current_device()
    plan = _plan(L, io, acc, config, dev)
    y = torch.empty_like(u, memory_format=torch.contiguous_format)
    plan.conv(u.contiguous(), Kf.contiguous(), y, stream=torch.cuda.current_stream(u.device))
    return y


@conv.register_fake
def _(u: Tensor, Kf: Tensor, acc: str = "fp32", config: str = "") -> Tensor:
    return torch.empty_like(u, memory_format=torch.contiguous_format)


def causal_conv(u: Tensor, k: Tensor, acc: str = "fp32", config: str = "") -> Tensor:
    """y[b,h,n] = sum_{m<=n} u[b,h,m] k[h,n-m]: the spectrum of k, then the fused convolution."""
    return conv(u, filter_spectrum(k, config), acc, config)


def two_sided_conv(u: Tensor, k: Tensor, acc: str = "fp32", config: str = "") -> Tensor:
    """Non-causal: y[b,h,n] = sum_{m<L} u[b,h,m] k[h,L-1+n-m] for k [H][2L-1] (k[:, L-1] is lag 0)."""
    return conv(u, filter_spectrum(k, config, "two_sided"), acc, config)


def circular_conv(u: Tensor, k: Tensor, acc: str = "fp32", config: str = "") -> Tensor:
    """Period-L circular: y[b,h,n] = sum_{m<L} u[b,h,m] k[h,(n-m) mod L] for k [H][L]."""
    return conv(u, filter_spectrum(k, config, "circular"), acc, config)


def _fft_plan(N: int, config: str, device) -> "sf.Plan":
    if N < 256 or N & (N - 1):
        raise ValueError("the transform length must be a power of two from 256 to 32768")
    dev = device.index if device.index is not None else torch.cuda.current_device()
    return _plan(N // 2, "fp32", "fp32", config, dev)


@torch.library.custom_op("sffft::rfft", mutates_args=())
def rfft(x: Tensor, config: str = "") -> Tensor:
    """Real DFT along the last axis (numpy.fft.rfft), fp32 with exact twiddles."""
    _check_cuda(x, "rfft")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("x must be float32 or bfloat16")
    plan = _fft_plan(x.shape[-1], config, x.device)
    return plan.rfft(x.contiguous(), stream=torch.cuda.current_stream(x.device))


@rfft.register_fake
def _(x: Tensor, config: str = "") -> Tensor:
    return x.new_empty(tuple(x.shape[:-1]) + (x.shape[-1] // 2 + 1,), dtype=torch.complex64)


@torch.library.custom_op("sffft::irfft", mutates_args=())
def irfft(X: Tensor, config: str = "") -> Tensor:
    """Inverse of rfft for an even length N = 2 (X.shape[-1] - 1) (numpy.fft.irfft)."""
    _check_cuda(X, "irfft")
    if X.dtype != torch.complex64:
        raise ValueError("X must be complex64")
    plan = _fft_plan(2 * (X.shape[-1] - 1), config, X.device)
    return plan.irfft(X.contiguous(), stream=torch.cuda.current_stream(X.device))


@irfft.register_fake
def _(X: Tensor, config: str = "") -> Tensor:
    return X.new_empty(tuple(X.shape[:-1]) + (2 * (X.shape[-1] - 1),), dtype=torch.float32)


# ---------------------------------------------------------------------------------------------------------------
# Linear attention and the norms around a block
# ---------------------------------------------------------------------------------------------------------------

@torch.library.custom_op("sffft::linear_attention", mutates_args=())
def _linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, initial_state: Optional[Tensor],
                      lengths: Optional[Tensor], scale: float) -> tuple[Tensor, Tensor]:
    return sf.linear_attention(q, k, v, log_decay, scale, initial_state, lengths)


@_linear_attention.register_fake
def _(q, k, v, log_decay, initial_state, lengths, scale):
    sf.check_linear_attention(q, k, v, log_decay, scale, initial_state, lengths)
    B, H, L, D = q.shape
    return sf._heads_like(q, B, H, L, v.shape[3], q.dtype), q.new_empty((B, H, D, v.shape[3]), dtype=torch.float32)


@torch.library.custom_op("sffft::linear_attention_backward", mutates_args=())
def _linear_attention_backward(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, initial_state: Optional[Tensor],
                               lengths: Optional[Tensor], scale: float, dy: Tensor,
                               dfinal_state: Optional[Tensor]) -> list[Tensor]:
    out = sf.linear_attention_backward(q, k, v, log_decay, dy, dfinal_state, scale, initial_state, lengths)
    return [t for t in out if t is not None]


@_linear_attention_backward.register_fake
def _(q, k, v, log_decay, initial_state, lengths, scale, dy, dfinal_state):
    out = [sf._heads_like(t, *t.shape, q.dtype) for t in (q, k, v)]
    return out if initial_state is None else out + [torch.empty_like(initial_state, memory_format=torch.contiguous_format)]


def _la_setup(ctx, inputs, output):
    q, k, v, log_decay, initial_state, lengths, scale = inputs
    ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths)
    ctx.scale = scale


def _la_backward(ctx, dy, dfinal_state):
    q, k, v, log_decay, initial_state, lengths = ctx.saved_tensors
    if dy is None:
        dy = q.new_zeros((*q.shape[:3], v.shape[3]))
    out = torch.ops.sffft.linear_attention_backward(q, k, v, log_decay, initial_state, lengths, ctx.scale, dy, dfinal_state)
    return out[0], out[1], out[2], None, out[3] if initial_state is not None else None, None, None


_linear_attention.register_autograd(_la_backward, setup_context=_la_setup)


def _eager(*tensors) -> bool:
    """Whether the tensors are plain CUDA tensors outside of any trace: the call then goes straight to the C ABI, which saves
    the operator's dispatch (tens of microseconds, and some hundreds with a gradient)."""
    if torch.compiler.is_compiling():
        return False
    return all(t is None or type(t) in (Tensor, torch.nn.Parameter) and t.is_cuda for t in tensors)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, lengths, scale):
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return sf.linear_attention(q, k, v, log_decay, scale, initial_state, lengths)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal_state):
        q, k, v, log_decay, initial_state, lengths = ctx.saved_tensors
        if dy is None:
            dy = q.new_zeros((*q.shape[:3], v.shape[3]))
        dq, dk, dv, ds = sf.linear_attention_backward(q, k, v, log_decay, dy, dfinal_state, ctx.scale, initial_state, lengths)
        return dq, dk, dv, None, ds, None, None


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, scale: float = 1.0,
                     initial_state: Optional[Tensor] = None, lengths: Optional[Tensor] = None) -> tuple[Tensor, Tensor]:
    """(y, final_state) of S_n = lambda S_{n-1} + k_n v_n^T, y_n = scale S_n^T q_n with lambda = exp(log_decay) for each
    head (see sffft_b200.linear_attention).  Differentiable in q, k, v and initial_state."""
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant: it has no gradient (pass log_decay.detach())")
    if _eager(q, k, v, log_decay, initial_state, lengths):
        if _wants_grad(q, k, v, initial_state):
            return _LinearAttention.apply(q, k, v, log_decay, initial_state, lengths, scale)
        return sf.linear_attention(q, k, v, log_decay, scale, initial_state, lengths)
    return _linear_attention(q, k, v, log_decay, initial_state, lengths, scale)


@torch.library.custom_op("sffft::linear_attention_step", mutates_args=("state",))
def _linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, slots: Optional[Tensor],
                           scale: float) -> Tensor:
    return sf.linear_attention_step(q, k, v, log_decay, state, slots, scale)


@_linear_attention_step.register_fake
def _(q, k, v, log_decay, state, slots, scale):
    return q.new_empty((q.shape[0], q.shape[1], v.shape[2]))


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, slots: Optional[Tensor] = None,
                          scale: float = 1.0) -> Tensor:
    """One token for each row, state[slot] updated in place (see sffft_b200.linear_attention_step).  No gradient."""
    if _wants_grad(q, k, v, log_decay, state):
        raise ValueError("linear_attention_step updates its state in place and has no gradient: use linear_attention, or no_grad")
    if _eager(q, k, v, log_decay, state, slots):
        return sf.linear_attention_step(q, k, v, log_decay, state, slots, scale)
    return _linear_attention_step(q, k, v, log_decay, state, slots, scale)


@torch.library.custom_op("sffft::block_norm", mutates_args=())
def _block_norm(x: Optional[Tensor], y: Optional[Tensor], gate: Optional[Tensor], post_weight: Optional[Tensor],
                weight: Optional[Tensor], scale: float, eps: float, groups: int, act: str, dim: int) -> list[Tensor]:
    """h (with y), n (with weight), then the rstd of y's groups (with post_weight) and of h (with weight)."""
    h, n, r1, r2 = sf.block_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, dim, stats=True)
    return [t for t in (None if y is None else h, n, r1, r2) if t is not None]


@_block_norm.register_fake
def _(x, y, gate, post_weight, weight, scale, eps, groups, act, dim):
    C, _, _ = sf.check_block_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
    lead = y if y is not None else x
    rows = lead.numel() // C
    out = []
    if y is not None:
        out.append(lead.new_empty(lead.shape, dtype=lead.dtype if x is None else x.dtype))
    if weight is not None:
        out.append(lead.new_empty(lead.shape))
    if post_weight is not None:
        out.append(lead.new_empty((rows, groups), dtype=torch.float32))
    if weight is not None:
        out.append(lead.new_empty((rows,), dtype=torch.float32))
    return out


@torch.library.custom_op("sffft::block_norm_backward", mutates_args=())
def _block_norm_backward(dh: Optional[Tensor], dn: Optional[Tensor], x: Optional[Tensor], y: Optional[Tensor],
                         gate: Optional[Tensor], post_weight: Optional[Tensor], weight: Optional[Tensor],
                         rstd_post: Optional[Tensor], rstd: Optional[Tensor], scale: float, eps: float, groups: int, act: str,
                         dim: int) -> list[Tensor]:
    out = sf.block_norm_backward(dh, dn, x, y, gate, post_weight, weight, rstd_post, rstd, scale, eps, groups, act, dim)
    return [t for t in out if t is not None]


@_block_norm_backward.register_fake
def _(dh, dn, x, y, gate, post_weight, weight, rstd_post, rstd, scale, eps, groups, act, dim):
    return [t.new_empty(t.shape) for t in (x, y, gate, post_weight, weight) if t is not None]


def _bn_setup(ctx, inputs, output):
    x, y, gate, post_weight, weight, *rest = inputs
    ctx.rest = rest
    kept = list(output)
    rstd = kept.pop() if weight is not None else None
    rstd_post = kept.pop() if post_weight is not None else None
    ctx.save_for_backward(x, y, gate, post_weight, weight, rstd_post, rstd)


def _bn_backward(ctx, grads):
    x, y, gate, post_weight, weight, rstd_post, rstd = ctx.saved_tensors
    grads = list(grads)
    lead = y if y is not None else x
    dh = grads.pop(0) if y is not None else None
    dn = grads.pop(0) if weight is not None else None
    if weight is not None and dn is None:
        dn = lead.new_zeros(lead.shape)
    if weight is None and dh is None:
        dh = lead.new_zeros(lead.shape, dtype=lead.dtype if x is None else x.dtype)
    out = torch.ops.sffft.block_norm_backward(dh, dn, x, y, gate, post_weight, weight, rstd_post, rstd, *ctx.rest)
    out = list(out)
    return tuple(out.pop(0) if t is not None else None for t in (x, y, gate, post_weight, weight)) + (None,) * 5


_block_norm.register_autograd(_bn_backward, setup_context=_bn_setup)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post_weight, weight, *rest):
        h, n, rstd_post, rstd = sf.block_norm(x, y, gate, post_weight, weight, *rest, stats=True)
        ctx.save_for_backward(x, y, gate, post_weight, weight, rstd_post, rstd)
        ctx.rest = rest
        ctx.set_materialize_grads(False)
        return None if y is None else h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        x, y, gate, post_weight, weight, rstd_post, rstd = ctx.saved_tensors
        lead = y if y is not None else x
        if weight is not None and dn is None:
            dn = torch.zeros_like(lead)
        if weight is None and dh is None:
            dh = torch.zeros_like(lead, dtype=lead.dtype if x is None else x.dtype)
        return (*sf.block_norm_backward(dh, dn, x, y, gate, post_weight, weight, rstd_post, rstd, *ctx.rest), *(None,) * 5)


def block_norm(x: Optional[Tensor] = None, y: Optional[Tensor] = None, gate: Optional[Tensor] = None,
               post_weight: Optional[Tensor] = None, weight: Optional[Tensor] = None, scale: float = 1.0, eps: float = 1e-6,
               groups: int = 1, act: str = "none", dim: int = -1) -> tuple[Tensor, Optional[Tensor]]:
    """(h, n) with a = y rstd_g(y) post_weight, h = x + scale act(gate) a, n = h rstd(h) weight: the norms before and after a
    block with its gate and residual scale (see sffft_b200.block_norm).  Differentiable in all its tensors."""
    if _eager(x, y, gate, post_weight, weight):
        if not _wants_grad(x, y, gate, post_weight, weight):
            return sf.block_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
        if y is None:
            return x, _BlockNorm.apply(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)[1]
        return _BlockNorm.apply(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
    out = _block_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
    h = x if y is None else out[0]
    return h, None if weight is None else out[0 if y is None else 1]
