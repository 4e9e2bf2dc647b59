"""A small language model on the package's operators, as an example of their use together.

Token ids are embedded (``embedding``), run through a ``HeadStartLSTM`` layer and gated recurrences
(``gated_recurrence``), and projected on the vocabulary; the log probabilities of the next tokens
(``token_logprobs``) are the training loss and what a server answers with.  ``step`` takes one token of
each of a batch of streams and updates their state in place.

``python -m prlstm_amd.language_model`` trains one on walks around a circle and continues them.
"""

import torch
import torch.nn as nn

from . import HeadStartLSTM
from .lm import embedding, gated_recurrence, gated_recurrence_step, token_logprobs


class GatedLayer(nn.Module):
    """``x + gated_recurrence(project(normalise(x)))``: gates of about 0.88 at first."""

    def __init__(self, width):
        super().__init__()
        self.norm = nn.LayerNorm(width)
        self.project = nn.Linear(width, 2 * width)
        with torch.no_grad():
            self.project.bias.zero_()
            self.project.bias[:width] = 2.0

    def forward(self, x, h0=None, reset=None):
        out, h = gated_recurrence(self.project(self.norm(x)), h0, reset)
        return x + out, h

    def step(self, x, h, reset=None):
        out, _ = gated_recurrence_step(self.project(self.norm(x)), h, reset, h_out=h)
        return x + out


class LanguageModel(nn.Module):
    """Next-token model over time-major ids [T, B].  A negative id is a padded position: its
    embedding is zero and it is not scored."""

    def __init__(self, vocab, width, layers=2, parallel=True):
        super().__init__()
        self.vocab, self.width = vocab, width
        self.weight = nn.Parameter(torch.randn(vocab, width) * width ** -0.5)
        self.lstm = HeadStartLSTM(width, width, parallel=parallel)
        self.layers = nn.ModuleList(GatedLayer(width) for _ in range(layers))
        self.norm = nn.LayerNorm(width)
        self.head = nn.Linear(width, vocab)

    def state(self, batch):
        """The state of ``batch`` new streams: the LSTM's (h, c) and each gated layer's, in fp32."""
        like = dict(dtype=torch.float32, device=self.weight.device)
        zeros = lambda: torch.zeros(batch, self.width, **like)  # noqa: E731
        return (zeros(), zeros()), [zeros() for _ in self.layers]

    def logits(self, x):
        return self.head(self.norm(x))

    def run_lstm(self, x, h, c, reset):
        """The LSTM over x from (h, c).  It has no reset of its own, so the sequence is run in parts
        that begin at the steps where a row has one (which the host reads)."""
        starts = [] if reset is None else reset.any(1).nonzero()[:, 0].tolist()
        if not starts:
            y, (h, c) = self.lstm(x, (h, c))
            return y, h[0], c[0]
        parts, bounds = [], [0, *(t for t in starts if t > 0), len(x)]
        for t0, t1 in zip(bounds, bounds[1:]):
            keep = ~reset[t0].bool()[:, None]
            h, c = (torch.where(keep, s, torch.zeros_like(s)) for s in (h, c))
            y, (h, c) = self.lstm(x[t0:t1], (h, c))
            h, c = h[0], c[0]
            parts.append(y)
        return torch.cat(parts), h, c

    def forward(self, ids, state=None, reset=None):
        """(logits [T, B, V], the state behind them).  Where ``reset`` [T, B] is set a new document
        begins: nothing of any layer's state passes."""
        (h, c), gated = self.state(ids.shape[1]) if state is None else state
        x = embedding(ids, self.weight, scale=self.width ** 0.5)
        y, h, c = self.run_lstm(x, h.to(x.dtype), c.to(x.dtype), reset)
        x = x + y
        after = []
        for layer, h0 in zip(self.layers, gated):
            x, h1 = layer(x, h0, reset)
            after.append(h1)
        return self.logits(x), ((h.float(), c.float()), after)

    def loss(self, ids, targets, reset=None):
        """Mean negative log probability of targets [T, B] (negative: not scored)."""
        logits, _ = self(ids, reset=reset)
        scored = (targets >= 0).sum().clamp_min(1)
        return -token_logprobs(logits, targets).logp.sum() / scored

    @torch.no_grad()
    def step(self, ids, state, top=0):
        """One token ids [B] of each stream: ``token_logprobs`` of the next one's logits.  The state
        is updated in place."""
        (h, c), gated = state
        x = embedding(ids, self.weight, scale=self.width ** 0.5)
        y, (h1, c1) = self.lstm(x[None], (h.to(x.dtype), c.to(x.dtype)))
        h.copy_(h1[0])
        c.copy_(c1[0])
        x = x + y[0]
        for layer, g in zip(self.layers, gated):
            x = layer.step(x, g)
        return token_logprobs(self.logits(x), top=top)


def main(steps=120, vocab=64, width=128, length=48, batch=32, device="cuda"):
    """Trains on walks around a fixed circle of the tokens, forwards or backwards as each began;
    returns the first and the last loss and the share of the next tokens that is right."""
    torch.manual_seed(0)
    model = LanguageModel(vocab, width).to(device)
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    g = torch.Generator().manual_seed(1)

    circle = torch.randperm(vocab, generator=g)

    def sequences():
        start, way = (torch.randint(0, n, (batch,), generator=g) for n in (vocab, 2))
        return circle[(start + torch.arange(length)[:, None] * (2 * way - 1)) % vocab].to(device)

    losses = []
    for _ in range(steps):
        ids = sequences()
        loss = model.loss(ids[:-1], ids[1:])
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    ids = sequences()
    state, right = model.state(batch), []
    for t in range(length - 1):
        best = model.step(ids[t], state, top=1).top_ids[:, 0]
        right.append((best == ids[t + 1]).float().mean())
    share = torch.stack(right[1:]).mean()  # two tokens show which way it goes
    return losses[0].item(), losses[-1].item(), share.item()


if __name__ == "__main__":
    first, last, share = main()
    print(f"loss {first:.3f} -> {last:.3f}; {100 * share:.0f}% of the next tokens right")
