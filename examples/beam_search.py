"""A small language model on linear attention with one decay a head: trained, prompted and searched.

    python examples/beam_search.py [--steps 60] [--beams 4] [--new 12]

The model (random weights, synthetic text: runs of a repeating pattern) is trained with chunk_decay for a few steps.  Prompts of different
lengths are then read in one ragged call, whose final states go into a beam search: each step is one decay_step a layer, from the states of the
beams that beam_select kept.  At the end the found sequences are scored again by chunk_decay over their whole length.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from gla_jax_amd import beam_select, chunk_decay, decay_step, reorder_states  # noqa: E402

F = torch.nn.functional


class Layer(torch.nn.Module):
    """Queries, keys and values of one projection; four heads to two key heads; a decay for each head and token."""

    def __init__(self, width, heads=4, key_heads=2, dk=32, dv=32):
        super().__init__()
        self.shape = heads, key_heads, dk, dv
        self.split = [key_heads * dk, key_heads * dk, heads * dv]
        self.project = torch.nn.Linear(width, sum(self.split), bias=False)
        self.decay = torch.nn.Linear(width, heads)
        self.back = torch.nn.Linear(heads * dv, width, bias=False)
        self.mix = torch.nn.Sequential(torch.nn.RMSNorm(width), torch.nn.Linear(width, 4 * width), torch.nn.SiLU(), torch.nn.Linear(4 * width, width))
        self.norm = torch.nn.RMSNorm(width)

    def rows(self, x):
        heads, key_heads, dk, dv = self.shape
        x = self.norm(x)
        q, k, v = self.project(x).split(self.split, -1)
        a = F.logsigmoid(self.decay(x).float() + 4.0)
        return a, v.unflatten(-1, (heads, dv)), F.normalize(k.unflatten(-1, (key_heads, dk)), dim=-1), q.unflatten(-1, (key_heads, dk))

    def state(self, batch, device):
        heads, _, dk, dv = self.shape
        return torch.zeros(batch, heads, dk, dv, device=device)

    def finish(self, x, out):
        x = x + self.back(out.flatten(-2))
        return x + self.mix(x)

    def forward(self, x, state, lengths=None):
        """[B,T,width] and the states before; what follows, and the states after."""
        state, out = chunk_decay(state, *self.rows(x), lengths)
        return self.finish(x, out), state

    def step(self, x, states, parents):
        """One token of every beam, [B,width]; `states` is updated where it lies."""
        return self.finish(x, decay_step(states, *self.rows(x), parents=parents))


class Model(torch.nn.Module):
    def __init__(self, vocab, width=64, layers=2):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width)
        self.layers = torch.nn.ModuleList(Layer(width) for _ in range(layers))
        self.head = torch.nn.Linear(width, vocab)

    def forward(self, tokens, lengths=None):
        x, states = self.embed(tokens), []
        for layer in self.layers:
            x, s = layer(x, layer.state(tokens.shape[0], tokens.device), lengths)
            states.append(s)
        return self.head(x), states

    def step(self, tokens, states, parents):
        x = self.embed(tokens)
        for layer, s in zip(self.layers, states):
            x = layer.step(x, s, parents)
        return self.head(x)


def text(batch, length, vocab, device, generator):
    """Patterns of 3 to 6 tokens, each repeated to the end."""
    rows = []
    for _ in range(batch):
        n = int(torch.randint(3, 7, (), generator=generator))
        pattern = torch.randint(3, vocab, (n,), generator=generator)
        rows.append(pattern.repeat(length // n + 1)[:length])
    return torch.stack(rows).to(device)


def search(model, prompts, lengths, beams, new, eos=2):
    """The best `beams` continuations of every prompt: tokens [G,W,new], scores [G,W], best first."""
    G, W = prompts.shape[0], beams
    with torch.no_grad():
        logits, states = model(prompts, lengths)
        # every beam starts from its prompt's state, and all but the first without a chance
        states = [s.repeat_interleave(W, 0) for s in states]
        logits = logits[torch.arange(G, device=prompts.device), lengths - 1][:, None].expand(G, W, -1)
        scores = torch.full((G, W), -float("inf"), device=prompts.device)
        scores[:, 0] = 0.0
        finished = torch.zeros(G, W, dtype=torch.bool, device=prompts.device)
        found = torch.zeros(G, W, 0, dtype=torch.int64, device=prompts.device)
        for _ in range(new):
            scores, parents, tokens = beam_select(logits, scores, finished=finished, eos=eos)
            finished = finished.gather(1, parents) | (tokens == eos)
            found = torch.cat([reorder_states(found.flatten(0, 1), parents).view(found.shape), tokens[..., None]], -1)
            logits = model.step(tokens.flatten(), states, parents).unflatten(0, (G, W))
    return found, scores


def main(steps=60, beams=4, new=12, vocab=40, seed=0):
    torch.manual_seed(seed)
    generator = torch.Generator().manual_seed(seed)
    model = Model(vocab).cuda()
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    first = last = None
    for i in range(steps):
        tokens = text(32, 96, vocab, "cuda", generator)
        logits, _ = model(tokens[:, :-1])
        loss = F.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        last = float(loss.detach())
        first = last if first is None else first
        if i % 20 == 0 or i == steps - 1:
            print(f"step {i}: loss {last:.3f}", flush=True)
    prompts = text(5, 33, vocab, "cuda", generator)
    lengths = torch.tensor([33, 20, 9, 26, 14], device="cuda", dtype=torch.int32)
    found, scores = search(model, prompts, lengths, beams, new)
    # the same sequences over their whole length
    again = torch.full_like(scores, 0.0)
    with torch.no_grad():
        for g in range(5):
            n = int(lengths[g])
            whole = torch.cat([prompts[g, :n].expand(beams, n), found[g]], -1)
            p = model(whole[:, :-1])[0].log_softmax(-1)[:, n - 1:].gather(-1, found[g][..., None])[..., 0]
            ended = (found[g] == 2).cumsum(-1) - (found[g] == 2).long() > 0         # after the end nothing counts
            again[g] = p.masked_fill(ended, 0.0).sum(-1)
            print("prompt", prompts[g, max(0, n - 7):n].tolist(), "->", found[g, 0].tolist(), f"score {float(scores[g, 0]):.3f}", flush=True)
    off = float((again - scores).abs().max())
    print(f"scores of the search and of the whole sequences differ by at most {off:.2e}")
    return first, last, off


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    for name, value in (("steps", 60), ("beams", 4), ("new", 12)):
        p.add_argument("--" + name, type=int, default=value)
    main(**vars(p.parse_args()))
