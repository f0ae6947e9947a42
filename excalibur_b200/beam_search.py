"""Beam search over a batch of sentences: every step's best continuations, and states that follow their beams.

    python -m excalibur_b200.beam_search [--sentences 2] [--beams 4] [--channels 512] [--vocab 8000] [--steps 12] [--experts 8] [--weights int8|e4m3]

searches with a small recurrent decoder of random weights (a feed-forward block by experts between an embedding and a vocabulary's weights in 8 bits) and
prints the best sequences.
"""
import argparse
import math

from . import capi


class BeamSearch:
    """Scores, tokens so far and which beams have ended, of sentences * beams rows."""

    def __init__(self, ctx, sentences, beams, end_token, most_tokens, temperature=1.0, device="cuda"):
        import torch
        self.ctx, self.sentences, self.beams, self.end_token, self.scale = ctx, sentences, beams, end_token, 1.0 / temperature
        self.scores = torch.full((sentences, beams), -math.inf, device=device)
        self.scores[:, 0] = 0.0                # the first step has one beam: all would go on alike
        self.ended = torch.zeros((sentences, beams), device=device, dtype=torch.bool)
        self.tokens = torch.full((sentences * beams, most_tokens), -1, device=device, dtype=torch.int32)
        self.length = 0

    def step(self, logits, states=(), lengths=None):
        """logits: (sentences * beams, vocabulary) of the next token; states: tensors (sentences * beams, ...) that follow the beams in place (lengths: as
        capi.reorder_beams takes them).  Returns the chosen tokens, (sentences * beams,) int32, -1 where there is no beam (its score is minus infinity)."""
        if self.length == self.tokens.shape[1]:
            raise ValueError("there is room for %d tokens" % self.length)
        scores, parents, chosen = capi.beam_select(self.ctx, logits, self.scores, scale=self.scale, ended=self.ended, end_token=self.end_token)
        if len(states):      # (the caller's first: where they are refused, nothing has changed)
            capi.reorder_beams(self.ctx, states, parents, lengths)
        capi.reorder_beams(self.ctx, self.tokens, parents)
        self.scores = scores
        self.tokens[:, self.length] = chosen.view(-1)
        self.length += 1
        self.ended = chosen == self.end_token      # (a beam that had ended goes on with that token)
        return chosen.view(-1)

    def finished(self):
        """Whether every beam has ended or is none (waits for the device)."""
        return bool((self.ended | (self.scores == -math.inf)).all())

    def best(self):
        """(tokens of every sentence's best beam, up to its end; their scores): a list of lists and a list."""
        rows = self.tokens.view(self.sentences, self.beams, -1)[:, 0, :self.length].tolist()      # (beams are in falling order)
        cut = [r[:r.index(self.end_token) + 1] if self.end_token in r else r for r in rows]
        return cut, self.scores[:, 0].tolist()


def main():
    import torch
    from .experts import Experts
    from .token_head import TokenHead
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--sentences", type=int, default=2)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--channels", type=int, default=512)
    p.add_argument("--vocab", type=int, default=8000)
    p.add_argument("--steps", type=int, default=12)
    p.add_argument("--experts", type=int, default=8)
    p.add_argument("--weights", choices=("int8", "e4m3"), default="int8")
    a = p.parse_args()
    ctx = capi.Context(torch.cuda.current_device())
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape):
        return torch.randn(shape, device="cuda", generator=gen)
    C, rows, k = a.channels, a.sentences * a.beams, min(2, a.experts)
    embedding, router = rand(a.vocab, C).half(), rand(a.experts, C).mul_(C ** -0.5).half()
    block = Experts(ctx, rand(a.experts, 2 * C, C).mul_(C ** -0.5).half(), rand(a.experts, C, 2 * C).mul_((2 * C) ** -0.5).half())
    head = TokenHead(ctx, rand(a.vocab, C).mul_(4 * C ** -0.5).half(), torch.ones(C, device="cuda"), weights=a.weights)
    search = BeamSearch(ctx, a.sentences, a.beams, end_token=0, most_tokens=a.steps)
    state = rand(a.sentences, C).half().repeat_interleave(a.beams, 0)
    for _ in range(a.steps):
        gates, chosen = torch.softmax((state @ router.t()).float(), 1).topk(k, 1)
        state, logits = head.logits(block(state, chosen, gates), state)
        tokens = search.step(logits, [state])
        if search.finished():
            break
        state = (0.5 * state + embedding[tokens.clamp_min(0).long()]).contiguous()
    ctx.sync_check()
    for i, (sequence, score) in enumerate(zip(*search.best())):
        print("sentence %d: %.3f, %s" % (i, score, " ".join(map(str, sequence))))


if __name__ == "__main__":
    main()
