"""The gated linear layer: in_proj -> gated linear recurrence -> out_proj.

The member of the family whose state enters linearly (no counterpart in the reference): with
f, c, z the thirds of in_proj(x),

    h_t = h_{t-1} + sigmoid(-f_t) (c_t - h_{t-1}),    y_t = h_t silu(z_t)

(elman_gated_linear_*), so that a sequence is scanned instead of walked.  Unlike the other layers' the
state is float32 in every dtype: with gates near one a 16-bit state would not move.  Document boundaries
inside a sequence are given as a reset mask.  LadderLM runs it as level "gated_linear".
"""
import torch
import torch.nn as nn

from . import fused_ops, hasty_pytorch_lib


class GatedLinearFunction(torch.autograd.Function):
    """forward(fcz [T,B,3d], h0 [B,d] | None, reset [T,B] | None) -> (y [T,B,d], h_last [B,d] float32);
    fcz is the projection as it comes, channels dense, any strides over t and b, and so is its gradient."""

    @staticmethod
    def forward(ctx, fcz, h0, reset):
        f, c, z = fcz.chunk(3, dim=-1)
        training = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        y, h_last, saved = hasty_pytorch_lib.gated_linear_forward(training, f, c, z, h0, reset)
        ctx.save_for_backward(fcz, saved, reset)
        ctx.set_materialize_grads(False)
        return y, h_last

    @staticmethod
    def backward(ctx, dy, dh_last):
        if torch.is_grad_enabled():      # create_graph: the result would silently be a constant
            raise RuntimeError("gated_linear: second derivatives are not supported")
        fcz, saved, reset = ctx.saved_tensors
        f, c, z = fcz.chunk(3, dim=-1)
        if dy is None:
            dy = torch.zeros_like(f)
        elif dy.shape[2] > 1 and dy.stride(2) != 1:
            dy = dy.contiguous()
        dfcz = hasty_pytorch_lib._sequence_like(fcz)
        *_, dh0 = hasty_pytorch_lib.gated_linear_backward(
            f, c, z, saved, dy, None if dh_last is None else dh_last.contiguous(), reset,
            out=dfcz.chunk(3, dim=-1))
        return dfcz, dh0 if ctx.needs_input_grad[1] else None, None


class GatedLinearElman(nn.Module):
    def __init__(self, dim, expansion=1.0, dropout=0.0, use_conv=False, mamba2_init=False, **kwargs):
        super().__init__()
        if use_conv:
            raise ValueError("GatedLinearElman has no convolution")
        self.dim = dim
        self.d_inner = int(dim * expansion)
        self.in_proj = nn.Linear(dim, 3 * self.d_inner, bias=True)
        self.out_proj = nn.Linear(self.d_inner, dim, bias=False)
        self.dropout = nn.Dropout(dropout) if dropout > 0 else nn.Identity()
        if mamba2_init:
            nn.init.normal_(self.in_proj.weight, std=0.02)
            nn.init.normal_(self.out_proj.weight, std=0.02)
        else:
            nn.init.xavier_uniform_(self.in_proj.weight)
            nn.init.xavier_uniform_(self.out_proj.weight)
        with torch.no_grad():      # memories from two steps to about four hundred
            self.in_proj.bias.zero_()
            self.in_proj.bias[:self.d_inner] = torch.linspace(0.0, 6.0, self.d_inner)

    def forward(self, x, h0=None, reset=None, **kwargs):
        """x: [B,T,dim], h0: [B,d_inner] float32, reset: [B,T] bool (True: this token starts a new document)
        -> (output [B,T,dim], h_final [B,d_inner] float32)."""
        if not fused_ops.library_handles(x):
            raise RuntimeError("elman_b200 runs on CUDA tensors (float32, bfloat16) only (no CPU fallback)")
        fcz = fused_ops.linear(x.contiguous(), self.in_proj.weight, self.in_proj.bias)
        y, h_final = fused_ops.gated_linear(fcz.transpose(0, 1), h0,
                                            None if reset is None else reset.t().contiguous())
        return fused_ops.linear(self.dropout(y.transpose(0, 1)).contiguous(), self.out_proj.weight), h_final

    def extra_repr(self):
        return f"dim={self.dim}, d_inner={self.d_inner}, LEVEL=GATED_LINEAR"
