"""Expert layers: tokens to their experts and back.

    rows, offsets, pos, src = sort_tokens(x, ids, experts)     # the rows of expert e are rows[offsets[e]:offsets[e + 1]]
    ...                                                        # any computation that keeps the rows in their places
    y = combine(rows, weights, pos, src)                       # y[t] = sum over j of weights[t, j] * rows[pos[t, j]]

Both have a gradient (no second one, no forward-mode derivative: both are refused) and neither waits for the device: shapes depend on the sizes,
not on the choices.  expert_linear multiplies the rows with their experts' kept int8 weights (serving); Int8MoE puts all of them together.
torch.jit.trace records each of them as a Python function.  The reference has no expert layers.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib as L
from . import kernels as K
from .linear import DEFAULT, Int8Config, Int8Linear, TokenLinearFn


def _once(name: str, inputs, *results):
    """The gradients have no gradient of their own: where a graph of them is made, going back through it is an error."""
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in inputs):
        return results
    error = torch._C._functions.DelayedError(f"trying to differentiate twice {name}, which has a first gradient only".encode(), 1)
    return tuple(None if r is None else error(r.detach().requires_grad_()) for r in results)


class _SortFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, experts, align):
        with K.untraced():
            rows, offsets, pos, src = K.sort_tokens(x, ids, experts, align)
        ctx.mark_non_differentiable(offsets, pos, src)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(pos)
        return rows, offsets, pos, src

    @staticmethod
    def backward(ctx, drows, *_):
        if drows is None:
            return None, None, None, None
        K.refuse_tangent("the gradient of sort_tokens", drows)
        dx = K.combine(drows.detach(), None, ctx.saved_tensors[0])   # a token's gradient is the sum of its rows'
        return *_once("sort_tokens", [drows], dx), None, None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, pos, src):
        with K.untraced():
            src = K._check_ints(src, "src", (rows.shape[0],))
            ctx.save_for_backward(rows, weights, pos, src)
            return K.combine(rows, weights, pos)

    @staticmethod
    def backward(ctx, dy):
        saved = ctx.saved_tensors
        K.refuse_tangent("the gradient of combine", dy)
        grads = K.combine_backward(*(t.detach() for t in saved), dy.detach(), ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return *_once("combine", [dy, *saved], *grads), None, None


def sort_tokens(x: torch.Tensor, ids: torch.Tensor, experts: int, align: int = 1):
    """x [T, H] (bf16, fp16, fp32), ids int32 or int64 [T, k], the experts of each token -> (rows, offsets, pos, src):

    rows [R, H]: a copy of x[t] for each choice ids[t, j], those of expert e from offsets[e] on in the order of (t, j).  offsets[e + 1]
    is the next multiple of `align` behind them (128: every segment is a whole number of blocks for Int8Linear).  Rows of no
    choice are zeros, also the ones from offsets[experts] on: R = sorted_rows(T, k, experts, align) covers any choices.
    pos int32 [T, k]: the row of a choice, or -1 where the id is outside [0, experts): such a choice is dropped (another rank's
    expert, or one above its capacity).  src int32 [R]: the inverse, t * k + j or -1.
    At most 1024 experts and 64 choices a token.  Gradient: that of x, summed in 32 bits."""
    if not torch.compiler.is_compiling():   # plain tensors: the same calls and autograd node without the interpreter
        done = K.host().sort_tokens(x, ids, experts, align)
        if done is not None:
            return done
    K.refuse_tangent("sort_tokens", x)
    K.refuse_proxies("sort_tokens")
    if torch.jit.is_tracing() or (torch.is_grad_enabled() and x.requires_grad):   # a trace records the function, not the launches
        return _SortFn.apply(x, ids, experts, align)
    return K.sort_tokens(x, ids, experts, align)


def combine(rows: torch.Tensor, weights: torch.Tensor, pos: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """rows [R, H], weights [T, k] (fp32 or the rows' type), pos and src of sort_tokens -> y [T, H] of the rows' type,
    y[t] = sum over j of weights[t, j] * rows[pos[t, j]], added in 32 bits and rounded once.  Dropped choices add nothing.
    Gradients: those of rows (zero for rows of no choice) and of weights (zero for dropped choices)."""
    if not torch.compiler.is_compiling():
        y = K.host().combine(rows, weights, pos, src)
        if y is not None:
            return y
    K.refuse_tangent("combine", rows, weights)
    K.refuse_proxies("combine")
    K._check_ints(src, "src", tuple(rows.shape[:1]))   # also where no gradient will need it
    if src.device != rows.device:
        raise ValueError(f"rows are on {rows.device}, src on {src.device}")
    if torch.jit.is_tracing() or (torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad)):
        return _CombineFn.apply(rows, weights, pos, src)
    return K.combine(rows, weights, pos)


def quantize_experts(weight: torch.Tensor):
    """weight bf16 [E, N, K] (or [N, K]), K a multiple of 128 -> (int8 of its shape, fp32 scales [E, N]): one scale an output channel,
    as double_channel quantizes it (triton/double-channle_fwd32.py:140-175)."""
    return K.quant_row(weight, L.QMODE_ROWRCP)


def expert_linear(rows: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, offsets: torch.Tensor, bias=None,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The experts' products for serving: rows bf16 [R, K] in the order of their experts, wq int8 [E, N, K] and ws fp32 [E, N]
    (quantize_experts), offsets int32 [E + 1] (sort_tokens), bias bf16 [E, N] -> [R, N], bf16 or fp32.  A row is quantized with
    one scale (an infinity makes its row NaN, a NaN counts as zero), the sum over K is exact, y = (sum * row scale) * channel scale +
    bias is rounded once.  Rows from offsets[E] on come out zero.  N a multiple of 8, K of 16; any number of rows, one included.
    The weights are integers, there is no gradient: inputs that want one are refused.  Int8Linear trains, on segments of
    sort_tokens(align=128)."""
    if out_dtype in (torch.bfloat16, torch.float32) and offsets is not None and not torch.compiler.is_compiling():
        y = K.host().token_linear(rows, wq, ws, offsets, bias, out_dtype == torch.float32)
        if y is not None:
            return y
    K.refuse_gradient("expert_linear", rows, ws, bias)
    if offsets is None:
        raise ValueError("expert_linear: offsets are needed (linear_w8a8 takes one matrix for all rows)")
    if torch.jit.is_tracing():
        return TokenLinearFn.apply(rows, wq, ws, offsets, bias, out_dtype)
    return K.token_linear(rows, wq, ws, offsets, bias, out_dtype)


def _biases(linears):
    """bf16 [len(linears), out_features], or None where no layer has one."""
    if all(m.bias is None for m in linears):
        return None
    return torch.stack([m.weight.new_zeros(m.weight.shape[0]) if m.bias is None else m.bias for m in linears]).to(torch.bfloat16)


def _thaw_loaded(module, keys) -> None:   # a function of the module's: the layer can be pickled
    module._thaw()


class Int8MoE(nn.Module):
    """Gated experts: y[t] = sum over the top_k experts e of token t of p_e * down_e(silu(gate_e(x)) * up_e(x)), p = softmax over the logits of
    the chosen ones.  hidden and mlp are multiples of 128.

    Training: the tokens are sorted with segments of whole blocks of 128 rows, and every expert's three linears are Int8Linear (or
    what `linear(in, out)` builds) on its segment; the sizes of the segments are read from the device once a forward pass.
    Serving: freeze() quantizes the weights once; forward passes without gradients then take expert_linear, any number of tokens from
    one on, without waiting for the device.  It is a copy of the weights as they are then: train(), load_state_dict() and moving
    the module drop it; after other changes to the weights freeze again."""

    def __init__(self, hidden: int, mlp: int, experts: int, top_k: int, device=None, config: Int8Config = DEFAULT, linear=None):
        super().__init__()
        if not 1 <= top_k <= experts:
            raise ValueError(f"top_k must be between 1 and the {experts} experts, got {top_k}")
        if linear is None:
            def linear(i, o):
                return Int8Linear(i, o, bias=False, device=device, config=config)
        self.experts, self.top_k = experts, top_k
        self.router = nn.Linear(hidden, experts, bias=False, device=device, dtype=torch.bfloat16)
        self.gate_proj = nn.ModuleList(linear(hidden, mlp) for _ in range(experts))
        self.up_proj = nn.ModuleList(linear(hidden, mlp) for _ in range(experts))
        self.down_proj = nn.ModuleList(linear(mlp, hidden) for _ in range(experts))
        self._frozen = None
        self.register_load_state_dict_post_hook(_thaw_loaded)

    def _thaw(self) -> None:
        self._frozen = None

    def _apply(self, fn, *args, **kwargs):   # to(), cuda(), half() and so on
        self._thaw()
        return super()._apply(fn, *args, **kwargs)

    @torch.no_grad()
    def freeze(self) -> "Int8MoE":
        gate_up = torch.stack([torch.cat([g.weight, u.weight]) for g, u in zip(self.gate_proj, self.up_proj)])
        down = torch.stack([d.weight for d in self.down_proj])
        bias = _biases([*self.gate_proj, *self.up_proj])
        if bias is not None:   # an expert's gate in front of its up, as their weights are
            bias = bias.view(2, self.experts, -1).transpose(0, 1).reshape(self.experts, -1)
        self._frozen = (*quantize_experts(gate_up), bias, *quantize_experts(down), _biases(self.down_proj))
        return self

    def train(self, mode: bool = True):
        if mode:
            self._thaw()
        return super().train(mode)

    def route(self, x: torch.Tensor):
        """x [T, hidden] -> (ids int64 [T, top_k], weights fp32 [T, top_k])."""
        logits, ids = self.router(x).float().topk(self.top_k, dim=-1)
        return ids, logits.softmax(-1)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x2 = x.reshape(-1, x.shape[-1])
        ids, weights = self.route(x2)
        if self._frozen is not None and not torch.is_grad_enabled():
            gate_up_q, gate_up_s, gate_up_b, down_q, down_s, down_b = self._frozen
            rows, offsets, pos, src = sort_tokens(x2, ids, self.experts)
            gate, up = expert_linear(rows, gate_up_q, gate_up_s, offsets, gate_up_b).chunk(2, -1)
            rows = expert_linear(F.silu(gate) * up, down_q, down_s, offsets, down_b)
        else:
            if torch.jit.is_tracing():
                raise RuntimeError("Int8MoE reads the sizes of its experts' segments from the device and a trace would keep them: trace a frozen "
                                   "layer (freeze()), without gradients")
            rows, offsets, pos, src = sort_tokens(x2, ids, self.experts, align=128)
            ends = offsets.tolist()
            parts = []
            for e, (a, b) in enumerate(zip(ends, ends[1:])):
                if b > a:
                    part = rows[a:b]
                    parts.append(self.down_proj[e](F.silu(self.gate_proj[e](part)) * self.up_proj[e](part)))
            rows = torch.cat([*parts, rows.new_zeros(rows.shape[0] - ends[-1], rows.shape[1])])
        return combine(rows, weights, pos, src).view(x.shape)
