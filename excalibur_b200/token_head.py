"""From a decoder's last hidden states to scores of tokens, with weights in 8 bits: the operators of ``capi`` that follow one another.

    python -m excalibur_b200.token_head [--rows 8] [--channels 1024] [--vocab 32000] [--top 5]

scores random hidden states with random weights and prints the most probable tokens of the first rows.
"""
import argparse

from . import capi


class TokenHead:
    """Norm weights, and a vocabulary's weights in e4m3 with a scale for each 128 x 128 of them."""

    def __init__(self, ctx, vocab_weights, norm_weight, post_weight=None, residual_scale=1.0, kind=capi.NORM_RMS, eps=1e-5):
        """vocab_weights: (tokens, channels) on the device, fp16, bf16 or fp32; norm weights: (channels,) fp32."""
        self.ctx, self.kind, self.eps, self.residual_scale = ctx, kind, eps, residual_scale
        self.norm_weight, self.post_weight = norm_weight, post_weight
        self.weights, self.scales = capi.quantize_blocks(ctx, vocab_weights, block_rows=128)

    def logits(self, h, x, gate=None, gate_rows=0, out_dtype=capi.EXB_F32):
        """The last block's result h (rows, channels) joins the residual stream x, and the norm of the sum is multiplied with the
        vocabulary.  Returns (residual stream, logits).  Logits are fp32 unless told otherwise: in fp16 one between 16 and 32 is off by up
        to 2^-7, its log probability with it, and one above 65504 is infinite."""
        r, q, s = capi.residual_norm(self.ctx, h, x, post_weight=self.post_weight, gate=gate, gate_rows=gate_rows, residual_scale=self.residual_scale,
                                     weight=self.norm_weight, kind=self.kind, eps=self.eps, quantized=True)
        return r, capi.fp8_matmul(self.ctx, q, s, self.weights, self.scales, out_dtype=out_dtype)

    def scores(self, h, x, tokens=None, top=0, temperature=1.0, **more):
        """(log probabilities of the given tokens, entropy, log probabilities of the `top` most probable tokens, those tokens)."""
        _, logits = self.logits(h, x, **more)
        return capi.token_logprobs(self.ctx, logits, tokens, top=top, scale=1.0 / temperature)


def main():
    import torch
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--rows", type=int, default=8)
    p.add_argument("--channels", type=int, default=1024)
    p.add_argument("--vocab", type=int, default=32000)
    p.add_argument("--top", type=int, default=5)
    a = p.parse_args()
    ctx = capi.Context(torch.cuda.current_device())
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape):
        return torch.randn(shape, device="cuda", generator=gen)
    head = TokenHead(ctx, rand(a.vocab, a.channels).mul_(3 * a.channels ** -0.5).half(), torch.ones(a.channels, device="cuda"))
    tokens = torch.randint(0, a.vocab, (a.rows, 1), device="cuda", generator=gen).int()
    given, entropy, best, best_tokens = head.scores(rand(a.rows, a.channels).half(), rand(a.rows, a.channels).half(), tokens, top=a.top)
    ctx.sync_check()
    for i in range(min(a.rows, 8)):
        print("row %d: token %d %.3f, entropy %.3f, best %s" % (
            i, int(tokens[i, 0]), float(given[i, 0]), float(entropy[i]), ", ".join("%d %.3f" % z for z in zip(best_tokens[i].tolist(), best[i].tolist()))))


if __name__ == "__main__":
    main()
