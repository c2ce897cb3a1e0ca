"""The feed-forward half of a decoder layer with experts, and an 8-bit projection on the same norm, on synthetic data.

  python examples/expert_layer.py [--tokens 48] [--layers 2]

For every layer: the attention's output is added to the residual stream and normed, in fp16 for the router and the experts and in
codes for a projection with 8-bit weights; a FullyConnected node scores the experts, tokens are routed to the best of them, and
their gated networks are weighted and added to the stream, in place.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def random_matrix(mld, gen, o, i, bits):
    """A quantised matrix of random weights: packed, scales, sums of the codes."""
    w = torch.randn(o, i, generator=gen, device="cuda") / i ** 0.5
    q, s = mld.quantize_weights(w, bits, 32 if bits == 4 else 0)
    packed, sums = mld.pack_weights(q, (o, 1, 1, i), bits, want_sum=True)
    return packed, mld.pack_scales(s, True), sums


class ExpertLayer:
    def __init__(self, mld, gen, width, ffn, experts, top_k, outputs, max_tokens):
        self.mld, self.width = mld, width
        self.norm = (1 + 0.1 * torch.randn(width, generator=gen, device="cuda")).half()
        rows = dict(src_layout=mld.LAYOUT_ROW_MAJOR, dst_layout=mld.LAYOUT_ROW_MAJOR, max_tokens=max_tokens)
        self.score = mld.FullyConnectedPlan(experts, width, 8, **rows)
        self.score_w = random_matrix(mld, gen, experts, width, 8)
        self.project = mld.FullyConnectedPlan(outputs, width, 8, prefill_act_quant=1, force_path=mld.PATH_GEMM, **rows)
        self.project_w = random_matrix(mld, gen, outputs, width, 8)
        self.router = mld.MoeRouter(experts, top_k, score=mld.MOE_SIGMOID, factor=1.5)
        self.balance = 0.01 * torch.randn(experts, generator=gen, device="cuda")
        self.experts = mld.MoeExperts(experts, top_k, width, ffn, max_tokens=max_tokens)
        each = [[random_matrix(mld, gen, 2 * ffn, width, 4) for _ in range(experts)], [random_matrix(mld, gen, width, ffn, 4) for _ in range(experts)]]
        self.weights = [torch.stack([m[i] for m in ms]) for ms in each for i in range(2)]
        new = lambda *shape, dtype=torch.float16: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
        self.y, self.logits, self.out = new(max_tokens, width), new(max_tokens, experts), new(max_tokens, outputs)
        self.codes, self.params = new(max_tokens, (width + 15) // 16 * 16, dtype=torch.int8), new(max_tokens, 3, dtype=torch.float32)
        self.ids, self.gates = new(max_tokens, top_k, dtype=torch.int32), new(max_tokens, top_k, dtype=torch.float32)

    def run(self, attention, stream):
        """attention, stream: fp16 [tokens][width]; the stream is updated in place.  Returns the projection's outputs."""
        n = stream.shape[0]
        y, codes, params, ids, gates = self.y[:n], self.codes[:n], self.params[:n], self.ids[:n], self.gates[:n]
        self.mld.add_rms_norm(attention, weight=self.norm, residual=stream, sum_out=stream, out=y, codes=codes, params=params)
        self.project.run_codes(codes, params, self.project_w[0], self.project_w[1], self.out, n)
        self.score.run(y, self.score_w[0], self.score_w[1], self.logits, n)
        self.router.run(self.logits[:n], ids, gates, bias=self.balance)
        self.experts.run(y, ids, gates, *self.weights, stream, residual=stream)
        return self.out[:n]


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--layers", type=int, default=2)
    args = ap.parse_args(argv)
    sys.path.insert(0, ROOT)
    import __graft_entry__ as g
    mld = g.import_package()
    gen = torch.Generator(device="cuda").manual_seed(0)
    layers = [ExpertLayer(mld, gen, 512, 256, 16, 4, 1024, args.tokens) for _ in range(args.layers)]
    stream = torch.randn(args.tokens, 512, generator=gen, device="cuda").half()
    for layer in layers:
        out = layer.run(torch.randn(args.tokens, 512, generator=gen, device="cuda").half(), stream)
        torch.cuda.synchronize()
        used = torch.unique(layer.ids[:args.tokens]).numel()
        print(f"{args.tokens} tokens over {used} experts, stream {stream.float().norm():.2f}, projection {out.float().norm():.2f}")
    return layers, stream


if __name__ == "__main__":
    main()
