"""A feed-forward block by experts: every token goes to a few of many pairs of matrices, in 8-bit integers or in the weights' own type."""
from . import capi


class Experts:
    """The weights of `experts` blocks x -> act(x up^T) down^T."""

    def __init__(self, ctx, up, down, weights="int8", act=capi.ACT_SILU):
        """up: (experts, hidden, channels), down: (experts, channels, hidden) on the device.  weights: "int8" (of fp16, bf16 or fp32 ones, with a scale
        for each expert's output channel), or "own": fp16 or bf16 as they are, with channels and hidden multiples of 8.  act: an activation of capi."""
        if weights not in ("int8", "own"):
            raise ValueError("weights are int8 or own, got %r" % (weights,))
        self.ctx, self.act, self.experts = ctx, act, up.shape[0]
        self.integers = weights == "int8"
        self.up, self.down = (self._laid_out(w) if self.integers else (w, None) for w in (up, down))

    def _laid_out(self, w):
        q, scales = capi.quantize_rows(self.ctx, w.reshape(-1, w.shape[2]))
        return q.unflatten(0, w.shape[:2]), scales.view(w.shape[:2])

    def _product(self, a, weights, ends, out_dtype):
        scales = None
        if self.integers:
            a, scales = capi.quantize_rows(self.ctx, a)
        return capi.grouped_matmul(self.ctx, a, weights[0], ends, scales, weights[1], out_dtype=out_dtype)

    def __call__(self, x, chosen, gates):
        """x: (rows, channels) fp16 (or the weights' own type); chosen: (rows, k) whole numbers below `experts`; gates: (rows, k).  Returns
        sum_j gates[:, j] * block[chosen[:, j]](x), in x's type."""
        import torch
        rows, k = chosen.shape
        order = chosen.reshape(-1).argsort(stable=True)                                          # places sorted by expert
        ends = (chosen.reshape(-1, 1) == torch.arange(self.experts, device=x.device)).sum(0).cumsum(0).int()
        out_dtype = capi.exb_dtype_of(x)
        h = self._product(x[order // k], self.up, ends, out_dtype)
        if h.dtype == torch.bfloat16:      # (the activations' kernels are for fp16 and fp32)
            h = capi.activation(self.ctx, h.float(), self.act).bfloat16()
        else:
            h = capi.activation(self.ctx, h, self.act)
        y = self._product(h, self.down, ends, capi.EXB_F32)
        each = torch.empty_like(y)
        each[order] = y
        return (each.view(rows, k, y.shape[1]) * gates.float()[..., None]).sum(1).to(x.dtype)
