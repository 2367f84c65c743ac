"""A small hybrid decoder on MI355X: delta-rule layers with a softmax-attention
layer after every few of them, trained on whole rows and served token by token.

The same weights run three ways through this package:

- ``train``: whole rows, ``chunk_gdn`` and ``causal_attention`` with rotary positions,
  differentiable; packed documents by ``segment_ids``;
- ``serve``: prompts of different length in one ragged batch over a paged cache
  (``paged_kv_append`` with the rotation, ``paged_attention``) and a carried delta-rule
  state per sequence;
- then one token per sequence and step (``gdn_decode_step``, the same two calls).

``python examples/hybrid_decoder.py`` runs a few training steps, serves two prompts
and compares each served token's logits with those of the whole row.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "deltanet-tpu_amd"))

from deltanet_tpu_amd import (  # noqa: E402
    apply_rotary, causal_attention, chunk_gdn, gdn_decode_step, paged_attention, paged_kv_append, rotary_table)


class DeltaLayer(torch.nn.Module):
    """Gated delta rule: one decay and one write strength per value head."""

    def __init__(self, width, Hk, Hv):
        super().__init__()
        self.Hk, self.Hv = Hk, Hv
        self.inp = torch.nn.Linear(width, (2 * Hk + Hv) * 128 + 2 * Hv, bias=False)
        self.out = torch.nn.Linear(Hv * 128, width, bias=False)

    def project(self, x):
        Hk, Hv = self.Hk, self.Hv
        q, k, v, a, b = self.inp(x).split([Hk * 128, Hk * 128, Hv * 128, Hv, Hv], dim=-1)
        heads = lambda t, h: F.silu(t).unflatten(-1, (h, 128))
        return heads(q, Hk), heads(k, Hk), heads(v, Hv), -F.softplus(a.float()), torch.sigmoid(b.float())

    def forward(self, x, seg):
        return self.out(chunk_gdn(*self.project(x), segment_ids=seg, qk_l2norm=True).flatten(2))

    def prompt(self, x, spans, states):
        """Ragged prompts (N, width); each sequence's state is kept."""
        outs = []
        for i, (a, b) in enumerate(spans):
            o, states[i:i + 1] = chunk_gdn(*(t[None] for t in self.project(x[a:b])), initial_state=states[i:i + 1],
                                           output_final_state=True, is_inference=True, qk_l2norm=True)
            outs.append(o[0])
        return self.out(torch.cat(outs).flatten(1))

    def token(self, x, states):
        o, new = gdn_decode_step(*self.project(x), states, qk_l2norm=True)
        states.copy_(new)
        return self.out(o.flatten(1))


class AttentionLayer(torch.nn.Module):
    """Grouped-query attention, a part of each head rotated by its position."""

    def __init__(self, width, Hq, Hkv, D):
        super().__init__()
        self.Hq, self.Hkv, self.D = Hq, Hkv, D
        self.inp = torch.nn.Linear(width, (Hq + 2 * Hkv) * D, bias=False)
        self.out = torch.nn.Linear(Hq * D, width, bias=False)

    def project(self, x):
        return self.inp(x).unflatten(-1, (-1, self.D)).split([self.Hq, self.Hkv, self.Hkv], dim=-2)

    def forward(self, x, seg, positions, table):
        q, k, v = self.project(x)
        q, k = apply_rotary(q, k, positions, table)
        return self.out(causal_attention(q, k, v, segment_ids=seg).flatten(2))

    def cached(self, x, positions, table, cache, pages, lens, cu):
        """New tokens (N, width) of all sequences: stored, then attended with what is there."""
        q, k, v = self.project(x)
        paged_kv_append(k, v, *cache, pages, lens, cu_seqlens=cu, table=table)
        q, _ = apply_rotary(q, None, positions, table)
        return self.out(paged_attention(q, *cache, pages, lens, cu_seqlens=cu).flatten(1))


class HybridDecoder(torch.nn.Module):
    def __init__(self, vocab=512, width=512, blocks=2, deltas=3, Hk=2, Hv=4, Hq=8, Hkv=2, D=128, rotary=64, most=4096, page=64):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width)
        self.layers = torch.nn.ModuleList()
        for _ in range(blocks):
            self.layers.extend(DeltaLayer(width, Hk, Hv) for _ in range(deltas))
            self.layers.append(AttentionLayer(width, Hq, Hkv, D))
        self.norms = torch.nn.ModuleList(torch.nn.RMSNorm(width) for _ in self.layers)
        self.head = torch.nn.Linear(width, vocab, bias=False)
        self.rotary, self.most, self.page = rotary, most, page

    def table(self):
        return rotary_table(self.most, self.rotary, device=self.head.weight.device)

    def forward(self, tokens, seg=None, positions=None):
        """Logits (B, L, vocab) of whole rows."""
        table = self.table()
        if positions is None:
            positions = torch.arange(tokens.shape[1], device=tokens.device)
        x = self.embed(tokens)
        for layer, norm in zip(self.layers, self.norms):
            y = norm(x)
            x = x + (layer(y, seg) if isinstance(layer, DeltaLayer) else layer(y, seg, positions, table))
        return self.head(x)

    @torch.no_grad()
    def serve(self, prompts, more):
        """Prompts (1D token tensors), then `more` (B, steps) given tokens one by one:
        the logits of each prompt's last token and of every later one, (B, steps + 1, vocab)."""
        dev, dt = self.head.weight.device, self.head.weight.dtype
        B, steps = more.shape
        n = [len(p) for p in prompts]
        per = [-(-(x + steps) // self.page) for x in n]
        pages = torch.zeros(B, max(per), dtype=torch.int32)
        for b, free in enumerate(torch.randperm(sum(per), dtype=torch.int32).split(per)):
            pages[b, :per[b]] = free
        pages, table = pages.to(dev), self.table()
        cu = torch.tensor([0] + n, dtype=torch.int32).cumsum(0).to(torch.int32)
        spans = list(zip(cu[:-1].tolist(), cu[1:].tolist()))
        cu, lens = cu.to(dev), torch.tensor(n, dtype=torch.int32, device=dev)
        state = []
        for layer in self.layers:
            if isinstance(layer, DeltaLayer):
                state.append(torch.zeros(B, layer.Hv, 128, 128, device=dev))
            else:
                shape = (sum(per), self.page, layer.Hkv, layer.D)
                state.append(tuple(torch.empty(shape, dtype=dt, device=dev) for _ in range(2)))

        def run(x, positions, cu, prompt):
            for layer, norm, s in zip(self.layers, self.norms, state):
                y = norm(x)
                if isinstance(layer, DeltaLayer):
                    x = x + (layer.prompt(y, spans, s) if prompt else layer.token(y, s))
                else:
                    x = x + layer.cached(y, positions, table, s, pages, lens, cu)
            return self.head(x)

        positions = torch.cat([torch.arange(x, device=dev) for x in n])
        logits = [run(self.embed(torch.cat(prompts)), positions, cu, True)[cu[1:].long() - 1]]
        for t in range(steps):
            lens += 1
            logits.append(run(self.embed(more[:, t]), lens - 1, None, False))
        return torch.stack(logits, dim=1)


def train_steps(model, steps=3, B=2, L=512, seed=0):
    """A few steps of next-token training on random packed documents; the losses."""
    dev = model.head.weight.device
    gen = torch.Generator(device=dev).manual_seed(seed)
    tokens = torch.randint(0, model.embed.num_embeddings, (B, L + 1), device=dev, generator=gen)
    start = torch.zeros(L, dtype=torch.int64, device=dev)
    start[L // 3:] = L // 3
    seg, positions = start.expand(B, L), torch.arange(L, device=dev) - start
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    losses = []
    for _ in range(steps):
        loss = F.cross_entropy(model(tokens[:, :-1], seg, positions).float().flatten(0, 1), tokens[:, 1:].flatten())
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return losses


@torch.no_grad()
def serving_error(model, lengths=(200, 77), steps=8, seed=1):
    """Relative difference (2-norms) of the served tokens' logits and the whole rows'."""
    dev = model.head.weight.device
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows = [torch.randint(0, model.embed.num_embeddings, (n + steps,), device=dev, generator=gen) for n in lengths]
    served = model.serve([r[:n] for r, n in zip(rows, lengths)], torch.stack([r[n:] for r, n in zip(rows, lengths)]))
    whole = torch.stack([model(r[None])[0, n - 1:] for r, n in zip(rows, lengths)])
    return float((served.float() - whole.float()).norm() / whole.float().norm())


def main():
    ap = argparse.ArgumentParser(description="A small hybrid decoder: training and paged serving")
    ap.add_argument("--dtype", choices=("bf16", "f32"), default="bf16")
    ap.add_argument("--steps", type=int, default=3)
    args = ap.parse_args()
    torch.manual_seed(0)
    model = HybridDecoder().to("cuda", torch.bfloat16 if args.dtype == "bf16" else torch.float32)
    print("losses", " ".join(f"{x:.4f}" for x in train_steps(model, args.steps)))
    print(f"served against whole rows: {serving_error(model):.2e}")


if __name__ == "__main__":
    main()
