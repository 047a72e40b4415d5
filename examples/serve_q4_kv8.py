"""Serving with the decode operators: prompts and then single tokens of a few
requests through a small Llama-shaped model with random Q4_0 weights and an
int8 paged cache.

    python examples/serve_q4_kv8.py [--layers 2] [--steps 8]

Each step: kv8_plan takes pages and gives the tokens their slots and positions;
in each layer the projections (ROCmEngine.matmul), kv8_append (keys rotated and
stored, queries rotated), kv8_attention; then sample.  Decode steps are captured
in a graph once and replayed: the lengths, tables and slots live on the device.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from ztensor_amd import storage as st  # noqa: E402
from ztensor_amd import synth  # noqa: E402
from ztensor_amd.decode import KV8Cache, rope_table  # noqa: E402
from ztensor_amd.engine import ROCmEngine  # noqa: E402


class Model:
    """Random weights in the shapes of a Llama layer; fp32 activations."""

    def __init__(self, engine: ROCmEngine, layers=2, hidden=1024, heads=8, kv_heads=2, dim=128, ffn=2816, vocab=4096, seed=1):
        self.e, self.heads, self.kv_heads, self.dim = engine, heads, kv_heads, dim
        g = torch.Generator().manual_seed(seed)
        self.embed = torch.randn(vocab, hidden, generator=g).to(engine.device)

        def weight(rows, k, n):
            w = synth.q4_0(rows, k, seed * 1000 + n)
            return st.Tensor((k, rows), st.Q4Storage.from_raw(w.raw, rows * k))  # [k, rows]: y = x @ w

        shapes = {"qkv": ((heads + 2 * kv_heads) * dim, hidden), "o": (hidden, heads * dim), "gate": (ffn, hidden),
                  "up": (ffn, hidden), "down": (hidden, ffn)}
        self.layers = [{name: weight(*s, 10 * i + j) for j, (name, s) in enumerate(shapes.items())} for i in range(layers)]
        self.head = weight(vocab, hidden, 999)
        self.table = rope_table(dim, 4096, base=500000.0, device=engine.device)

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)

    def caches(self, pages, page_tokens):
        return [KV8Cache.allocate(pages, self.kv_heads, self.dim, page_tokens, self.e.device) for _ in self.layers]

    def forward(self, tokens, plan, caches, max_q, max_kv):
        """The last hidden states of a step's tokens [tokens, hidden]."""
        e, x, t = self.e, self.embed[tokens], tokens.numel()
        split = [self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim]
        for w, cache in zip(self.layers, caches):
            q, k, v = (p.view(t, -1, self.dim) for p in e.matmul(self.norm(x), w["qkv"]).split(split, 1))
            q = e.kv8_append(k, v, cache, plan.slots, positions=plan.positions, table=self.table, q=q)
            a = e.kv8_attention(q, cache, plan.block_table, plan.kv_lens, plan.q_start, max_q=max_q, max_kv=max_kv)
            x = x + self.norm(e.matmul(a.view(t, -1), w["o"]))
            h = self.norm(x)
            f = torch.nn.functional.silu(self.norm(e.matmul(h, w["gate"]))) * self.norm(e.matmul(h, w["up"]))
            x = x + self.norm(e.matmul(f, w["down"]))
        return self.norm(x)


class Server:
    """The requests' state on the device, and a step over it."""

    def __init__(self, model: Model, requests: int, pages=64, page_tokens=64, width=16):
        self.m, self.page_tokens, self.width = model, page_tokens, width
        e = model.e
        i32 = {"dtype": torch.int32, "device": e.device}
        self.caches = model.caches(pages, page_tokens)
        self.lens, self.table = torch.zeros(requests, **i32), torch.full((requests, width), -1, **i32)
        self.free, self.free_count = torch.arange(pages, **i32), torch.tensor([pages], **i32)

    def step(self, tokens, new, max_q, max_kv):
        """Hidden states of `tokens`, new[r] of them of request r.  Where self.took[r] is false the pages did not suffice:
        the request's length stays, and its hidden states have no meaning."""
        p = self.m.e.kv8_plan(self.lens, new, self.table, self.free, self.free_count, self.page_tokens, tokens.numel(),
                              in_place=True)
        x = self.m.forward(tokens, p, self.caches, max_q, max_kv)
        self.took = p.kv_lens == self.lens + new
        self.lens.copy_(p.kv_lens)
        self.free_count.copy_(p.free_count)
        return x, p

    def release(self, r: int):
        """Ends request r: its pages go back to the free list."""
        n = -(-int(self.lens[r]) // self.page_tokens)
        at = int(self.free_count)
        self.free[at:at + n] = self.table[r, :n]
        self.free_count += n
        self.lens[r] = 0


def generate(engine, prompts, steps, layers=2, seed=1, pages=64, **sampling):
    """Tokens of each request: the prompts together, then one token of each a step; -1 in steps for which a request got
    no page (it goes on where it was once there is one)."""
    with torch.cuda.stream(engine.stream):
        model = Model(engine, layers=layers)
        r = len(prompts)
        server = Server(model, r, pages)
        most = max(map(len, prompts)) + steps
        dev = engine.device
        gen = torch.Generator(device=dev).manual_seed(seed)
        new = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
        x, p = server.step(torch.tensor(sum(prompts, []), device=dev), new, max(map(len, prompts)), most)
        if not bool(server.took.all()):
            raise RuntimeError(f"{pages} pages do not hold the prompts")
        logits = engine.matmul(x[p.q_start[1:].long() - 1], model.head)
        token, _ = engine.sample(logits, torch.rand(r, device=dev, generator=gen), **sampling)
        out, given = [token.clone()], token.clone()
        one = torch.ones(r, dtype=torch.int32, device=dev)
        u = torch.empty(r, device=dev)

        def decode():
            x, _ = server.step(token, one, 1, most)
            t, _ = engine.sample(engine.matmul(x, model.head), u, **sampling)
            given.copy_(torch.where(server.took, t, -1))
            token.copy_(torch.where(server.took, t, token))

        graph = None
        for i in range(steps - 1):
            u.copy_(torch.rand(r, device=dev, generator=gen))
            if graph is None and i == 1:  # the first step has made the weights' copies and the workspace
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=engine.stream):
                    decode()
            if graph is None:
                decode()
            else:
                graph.replay()
            out.append(given.clone())
        torch.cuda.synchronize()
        return model, server, torch.stack(out, 1)


def main():
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--layers", type=int, default=2)
    a.add_argument("--steps", type=int, default=8)
    a = a.parse_args()
    engine = ROCmEngine(stream=torch.cuda.Stream())
    prompts = [list(range(5, 5 + n)) for n in (3, 130, 64)]
    top_p = torch.full((3,), 0.9, device=engine.device)
    _, server, tokens = generate(engine, prompts, a.steps, a.layers, top_p=top_p)
    for p, t in zip(prompts, tokens.tolist()):
        print(f"{len(p)} tokens of prompt, then {t}")
    print("lengths", server.lens.tolist(), "free pages", int(server.free_count))


if __name__ == "__main__":
    main()
