"""Sequences served from a key/value cache in 4 bits: prompts in chunks, tokens one by one for all sequences at once, a
conversation that forks, pages moved together when sequences end.

A stack of attention layers (int4 projections, norms of queries and keys with the rotation, cache, attention, int4 projection
back, sum) stands for a model.  Everything that a step needs is queued on the current stream; the page tables are the host's.

    python examples/paged_serving.py [--layers 4] [--d-model 2048] [--prompt 700] [--steps 32]
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__  # noqa: E402

mld = __graft_entry__.import_package()


class Projection:
    """A linear layer held in 4 bits with a scale per 32 inputs."""

    def __init__(self, n, k, most, generator):
        w = torch.randn(n, k, generator=generator, device="cuda") / k ** 0.5
        codes, scale = mld.quantize_weights(w, 4, block=32)
        self.weights, _ = mld.pack_weights(codes, (n, 1, 1, k), 4, group=32)
        self.scale, self.n = mld.pack_scales(scale, True), n
        self.plan = mld.FullyConnectedPlan(n, k, 4, scale_mode=mld.SCALE_BLOCK, groups=k // 32, precision=mld.F32F16,
                                           src_layout=mld.LAYOUT_ROW_MAJOR, dst_layout=mld.LAYOUT_ROW_MAJOR, max_tokens=most)

    def __call__(self, x):
        y = torch.empty(x.shape[0], self.n, dtype=torch.float16, device="cuda")
        self.plan.run(x, self.weights, self.scale, y, x.shape[0])
        return y


class Server:
    def __init__(self, layers=2, d_model=1024, heads=16, kv_heads=4, head_dim=64, page_tokens=32, pages=256, max_batch=8,
                 most=512, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.most = heads, kv_heads, head_dim, most
        self.cache = mld.Kv4Cache(kv_heads, head_dim, page_tokens, pages, layers=layers)
        self.pager = mld.Kv4Pager(pages, page_tokens, max_batch)
        self.rope = mld.QkNormRope(heads, kv_heads, head_dim)
        self.attention = mld.Kv4Attention(self.cache, heads, max_batch, pages)
        self.tables = torch.zeros(max_batch, pages, dtype=torch.int32).pin_memory()
        self.layers = []
        for _ in range(layers):
            self.layers.append({
                "qkv": Projection((heads + 2 * kv_heads) * head_dim, d_model, most, g),
                "out": Projection(d_model, heads * head_dim, most, g),
                "norm": torch.rand(d_model, generator=g, device="cuda").half() + 0.5,
                "q_norm": torch.rand(head_dim, generator=g, device="cuda").half() + 0.5,
                "k_norm": torch.rand(head_dim, generator=g, device="cuda").half() + 0.5})

    def step(self, work):
        """work: [(sequence, x)], x the new tokens' vectors, fp16 [tokens][d_model].  Returns a tensor like x for each."""
        starts, slots, positions, lens = [0], [], [], []
        self.tables.zero_()
        for row, (sequence, x) in enumerate(work):
            begin = self.pager.length(sequence)
            new, copies = self.pager.append(sequence, x.shape[0])
            if copies:  # the last page is another sequence's too: it gets its own before it is written
                self.cache.copy_pages(*zip(*copies))
            slots += new
            positions += range(begin, begin + x.shape[0])
            starts.append(starts[-1] + x.shape[0])
            lens.append(begin + x.shape[0])
            table = self.pager.table(sequence)
            self.tables[row, :len(table)] = torch.tensor(table, dtype=torch.int32)
        n = starts[-1]
        device = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
        slots, positions, lens, q_starts = map(device, (slots, positions, lens, starts))
        tables = self.tables[:len(work)].cuda()
        longest = max(x.shape[0] for _, x in work)

        h, hk, d = self.heads, self.kv_heads, self.head_dim
        x = torch.cat([x for _, x in work])
        q = torch.empty(n, h, d, dtype=torch.float16, device="cuda")
        o = torch.empty_like(q)
        for number, layer in enumerate(self.layers):
            y = torch.nn.functional.rms_norm(x.float(), x.shape[1:], eps=1e-6).half() * layer["norm"]
            qkv = layer["qkv"](y).view(n, h + 2 * hk, d)
            self.rope.run(qkv[:, :h], qkv[:, h:h + hk], positions, q, q_weight=layer["q_norm"], k_weight=layer["k_norm"],
                          v=qkv[:, h + hk:], cache=self.cache, slots=slots, layer=number)
            self.attention.run(q, tables, lens, o, q_starts=q_starts, max_queries=longest, layer=number)
            x = x + layer["out"](o.view(n, h * d))
        return list(x.split([b - a for a, b in zip(starts, starts[1:])]))

    def prompt(self, sequence, x):
        """A prompt of any length, in chunks of at most `most` tokens."""
        return torch.cat([self.step([(sequence, part)])[0] for part in x.split(self.most)])

    def compact(self):
        """Moves pages into the places that ended sequences left, so that the pool's used part has no holes."""
        src, dst = self.pager.compact()
        if src:
            self.cache.copy_pages(src, dst)
        return len(src)

    def check(self):
        """Raises if a kernel found a page or a length out of range, or gave up waiting (waits for the stream)."""
        torch.cuda.synchronize()
        code = self.attention.device_status()
        if code:
            raise RuntimeError(f"attention: device status {code}")


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--d-model", type=int, default=2048)
    parser.add_argument("--prompt", type=int, default=700)
    parser.add_argument("--steps", type=int, default=32)
    args = parser.parse_args()
    pages = 4 * (-(-(args.prompt + args.steps) // 64) + 1)
    server = Server(args.layers, args.d_model, heads=args.d_model // 128, kv_heads=max(1, args.d_model // 512), head_dim=128,
                    page_tokens=64, pages=pages, max_batch=4)
    first, second = server.pager.open(), server.pager.open()
    last = [server.prompt(s, torch.randn(args.prompt // (1 + s), args.d_model, device="cuda").half())[-1:] for s in (first, second)]
    branch = server.pager.fork(first)  # the same conversation, continued in another way
    sequences, last = [first, second, branch], last + [torch.randn(1, args.d_model, device="cuda").half()]
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(args.steps):
        if step == min(3, args.steps - 1):
            begin.record()
        last = [y / y.float().square().mean().sqrt().half() for y in server.step(list(zip(sequences, last)))]
    end.record()
    server.check()
    timed = args.steps - min(3, args.steps - 1)
    print(f"{args.layers} layers, prompts of {args.prompt} and {args.prompt // 2}, {len(sequences)} sequences: "
          f"{begin.elapsed_time(end) / timed:.3f} ms a step")
    server.pager.close_sequence(second)
    print(f"second sequence ended: {server.compact()} pages moved, {server.pager.free_pages()} of {pages} free")
    server.step([(first, last[0]), (branch, last[2])])
    server.check()


if __name__ == "__main__":
    main()
