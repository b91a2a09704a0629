#!/usr/bin/env python3
"""Several requests through a small decoder with random weights, over a paged 4-bit latent cache: prompts of different
lengths in one step, then one token a request and step, one request forked on the way.

    python examples/serve_requests.py [--steps 16] [--seed 0]

Prints every request's tokens with their log probabilities and the mean log probability of its prompt. The decoder is
MLA attention in its absorbed form (glm.c infer.c:955-1085) with dense SwiGLU layers, in bf16 with torch's products.
"""
import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Decoder:
    """Random weights; q_a, the router and the experts are left out."""

    def __init__(self, layers=2, hidden=512, heads=8, nope=64, rope=64, kv_lora=256, v_dim=64, ffn=1024, vocab=5003, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device="cuda") / math.sqrt(shape[-2])).to(torch.bfloat16)

        self.layers, self.heads, self.nope, self.rope, self.kv_lora, self.vocab = layers, heads, nope, rope, kv_lora, vocab
        self.scale = 1 / math.sqrt(nope + rope)
        self.embed = torch.randn(vocab, hidden, generator=g, device="cuda").to(torch.bfloat16)
        self.lm_head = w(hidden, vocab) * 4
        self.w = [dict(q=w(hidden, heads * (nope + rope)), kv=w(hidden, kv_lora + rope), k_b=w(heads, nope, kv_lora),
                       v_b=w(heads, kv_lora, v_dim), o=w(heads * v_dim, hidden), up=w(hidden, 2 * ffn), down=w(ffn, hidden))
                  for _ in range(layers)]
        self.freq = 10000.0 ** (-torch.arange(rope // 2, device="cuda") / (rope // 2))

    def _rotate(self, x, pos):
        a = pos.view(-1, *[1] * (x.dim() - 1)) * self.freq
        lo, hi = x.float().chunk(2, -1)
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1).to(x.dtype)

    @staticmethod
    def _norm(x):
        return torch.nn.functional.rms_norm(x, x.shape[-1:], eps=1e-5)

    def forward(self, pool, step, tokens):
        """Logits [tokens, vocab] of the step's tokens."""
        x = self.embed[tokens]
        for i, w in enumerate(self.w):
            h = self._norm(x)
            q = (h @ w["q"]).view(-1, self.heads, self.nope + self.rope)
            kv = h @ w["kv"]
            pool.store(i, step, self._norm(kv[:, :self.kv_lora]), self._rotate(kv[:, self.kv_lora:], step.pos))
            absorbed = torch.einsum("thn,hnl->thl", q[..., :self.nope], w["k_b"])
            ctx = pool.attend(i, step, torch.cat([absorbed, self._rotate(q[..., self.nope:], step.pos)], -1), self.scale)
            x = x + torch.einsum("thl,hlv->thv", ctx, w["v_b"]).flatten(1) @ w["o"]
            gate, up = (self._norm(x) @ w["up"]).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ w["down"]
        return self._norm(x) @ self.lm_head


def serve(lib, pool_type, prompts, steps, fork_at=None, seed=0, page_size=16):
    """{request: dict(tokens, logprobs, prompt_logprob, alternatives)} of greedy decoding; with fork_at, request 0 is
    forked after that many steps, and the fork goes on with the second most likely token."""
    model = Decoder(seed=seed)
    most = max(map(len, prompts)) + steps
    pool = pool_type(lib, model.layers, (len(prompts) + 1) * -(-most // page_size), model.kv_lora, model.rope, page_size,
                     len(prompts) + 1, most)
    result = {}
    for r, p in enumerate(prompts):
        pool.open(r)
    # the prompts, in one step
    step = pool.plan({r: len(p) for r, p in enumerate(prompts)})
    flat = torch.tensor([t for p in prompts for t in p], device="cuda")
    logits = model.forward(pool, step, flat)
    target = torch.tensor([t for p in prompts for t in p[1:] + [-1]], dtype=torch.int32, device="cuda")
    told = pool.scores(logits, target)[0].tolist()  # -inf where nothing follows
    at = 0
    for r, p in enumerate(prompts):
        result[r] = dict(tokens=list(p), logprobs=[], alternatives=[], prompt=len(p), prompt_logprobs=told[at:at + len(p) - 1])
        at += len(p)
    logits = logits[step.last]
    for n in range(steps):
        order = step.requests
        _, _, ids, tops = pool.scores(logits, k=2)
        ids, tops = ids.tolist(), tops.tolist()
        if n == fork_at:
            new = len(prompts)
            pool.fork(0, new)
            result[new] = {k: v if k == "prompt" else list(v) for k, v in result[0].items()}
            order, ids, tops = order + [new], ids + [ids[0][::-1]], tops + [tops[0][::-1]]
        for r, i, lp in zip(order, ids, tops):
            result[r]["tokens"].append(i[0])
            result[r]["logprobs"].append(lp[0])
            result[r]["alternatives"].append((i[1], lp[1]))
        if n + 1 < steps:
            step = pool.plan({r: 1 for r in order})
            logits = model.forward(pool, step, torch.tensor([result[r]["tokens"][-1] for r in order], device="cuda"))
    return result, pool, model


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args()
    sys.path.insert(0, ROOT)
    from __graft_entry__ import load_package

    pkg = load_package()
    pkg.build.build()
    import importlib
    pool_type = importlib.import_module(pkg.__name__ + ".serve").LatentPool
    g = torch.Generator().manual_seed(args.seed)
    prompts = [torch.randint(5003, (n,), generator=g).tolist() for n in (1, 37, 200, 16)]
    result, _, _ = serve(pkg.glm_cuda.GlmCuda(), pool_type, prompts, args.steps, fork_at=args.steps // 2, seed=args.seed)
    for r, out in result.items():
        told = out["prompt_logprobs"]
        print(f"request {r}: prompt of {out['prompt']}, mean log probability "
              f"{sum(told) / len(told) if told else float('nan'):.3f}")
        print("   ", " ".join(f"{t}({lp:.2f})" for t, lp in zip(out["tokens"][out["prompt"]:], out["logprobs"])))


if __name__ == "__main__":
    main()
