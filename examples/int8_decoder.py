"""A small decoder's feed-forward side on the 8-bit integer operators, as a serving engine would run them.

    python examples/int8_decoder.py [--hidden 2048 --intermediate 768 --dense 8192 --experts 64 --top-k 8 --layers 4 --prompt 512 --steps 32]

Layers alternate between a dense MLP (residual add + norm + quantise, gate_up, SiLU * mul + quantise, down) and an expert layer; a head
projects the last token.  Weights are random, made in 16 bits and quantised on the GPU by the same operator that quantises tokens.  A prompt
runs eagerly, single-token steps as a replayed CUDA graph; the first step is compared with the same decoder in 32-bit floats and
unquantised weights.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "llm-scaler_b200"))
import custom_esimd_kernels_vllm as b2q  # noqa: E402

EPS = 1e-6


def norm(x, weight):
    return torch.nn.functional.rms_norm(x.float(), x.shape[-1:], weight.float(), EPS)


class Linear:
    """An int8 weight made from a float one; keeps the float one where it is to be compared."""

    def __init__(self, weight, keep):
        self.float = weight.float() if keep else None
        self.codes, self.scale = b2q.quantize_int8(weight)

    def __call__(self, codes, scale):
        return b2q.linear_int8(codes, scale, self.codes, self.scale)


class Dense:
    def __init__(self, make, hidden, inter, keep):
        self.norm = make(hidden) * 0.1 + 1
        self.gate_up, self.down = Linear(make(2 * inter, hidden), keep), Linear(make(hidden, inter), keep)

    def __call__(self, x, residual):
        """x: what the layer in front adds to residual, which is updated in place; returns this layer's contribution."""
        gate_up = self.gate_up(*b2q.resadd_rmsnorm_quantize_int8(x, residual, self.norm, EPS))
        return self.down(*b2q.silu_mul_quantize_int8(gate_up))

    def reference(self, x, residual):
        residual += x
        gate, up = (norm(residual, self.norm) @ self.gate_up.float.t()).chunk(2, -1)
        return (torch.nn.functional.silu(gate) * up) @ self.down.float.t()


class Experts:
    def __init__(self, make, hidden, inter, experts, top_k, keep):
        self.norm, self.top_k, self.hidden = make(hidden) * 0.1 + 1, top_k, hidden
        self.router = make(experts, hidden) * 4
        w13, w2 = make(experts, 2 * inter, hidden), make(experts, hidden, inter)
        self.float = (w13.float(), w2.float()) if keep else None
        c, s = b2q.quantize_int8(w13.flatten(0, 1))
        self.w13, self.s13 = c.view(w13.shape), s.view(experts, -1)
        c, s = b2q.quantize_int8(w2.flatten(0, 1))
        self.w2, self.s2 = c.view(w2.shape), s.view(experts, -1)

    def __call__(self, x, residual):
        residual += x
        normed = norm(residual, self.norm).to(x.dtype)
        self.logits = normed @ self.router.t()
        return b2q.moe_forward_int8(normed, self.logits, self.w13, self.s13, self.w2, self.s2, self.top_k)

    def reference(self, x, residual):
        """Takes the logits of the call in front, so that both choose the same experts."""
        residual += x
        normed = norm(residual, self.norm)
        top, ids = self.logits.float().topk(self.top_k)
        weights, out = top.softmax(-1), torch.zeros_like(normed)
        for t in range(len(x)):
            for w, e in zip(weights[t], ids[t].tolist()):
                gate, up = (self.float[0][e] @ normed[t]).chunk(2)
                out[t] += w * (self.float[1][e] @ (torch.nn.functional.silu(gate) * up))
        return out


class Decoder:
    def __init__(self, hidden, intermediate, dense, experts, top_k, layers, vocab, seed=0, keep=False, dtype=torch.bfloat16, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)

        def make(*shape):
            return (torch.randn(*shape, generator=g, device=device) / shape[-1] ** 0.5).to(dtype)

        self.layers = [Experts(make, hidden, intermediate, experts, top_k, keep) if i % 2 else Dense(make, hidden, dense, keep) for i in range(layers)]
        self.head = Linear(make(vocab, hidden), keep)
        self.embedding = torch.randn(vocab, hidden, generator=g, device=device).to(dtype)

    def __call__(self, tokens):
        """Logits of the last of tokens (int64 [T])."""
        residual = self.embedding[tokens]
        x = torch.zeros_like(residual)
        for layer in self.layers:
            x = layer(x, residual)
        return b2q.linear_int8_dynamic((residual + x)[-1:], self.head.codes, self.head.scale)

    def reference(self, tokens):
        residual = self.embedding[tokens].float()
        x = torch.zeros_like(residual)
        for layer in self.layers:
            x = layer.reference(x, residual)
        return (residual + x)[-1:] @ self.head.float.t()


def capture(decoder, token):
    """A graph of one step: reads token, writes the logits and, into token, the choice."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        decoder(token)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = decoder(token)
        token.copy_(logits.argmax(-1))
    return graph, logits


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("hidden", 2048), ("intermediate", 768), ("dense", 8192), ("experts", 64), ("top-k", 8), ("layers", 4), ("vocab", 32000), ("prompt", 512), ("steps", 32), ("seed", 0)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    decoder = Decoder(a.hidden, a.intermediate, a.dense, a.experts, a.top_k, a.layers, a.vocab, a.seed, keep=True)
    torch.cuda.synchronize()
    b2q.set_overlap_mode(2)      # no weight is written from here on
    prompt = torch.randint(a.vocab, (a.prompt,), generator=torch.Generator("cuda").manual_seed(a.seed), device="cuda")

    first = decoder(prompt)
    token = first.argmax(-1)
    eager = decoder(token).float()
    exact = decoder.reference(token)
    error = float((eager - exact).norm() / exact.norm())
    graph, logits = capture(decoder, start := token.clone())
    graph.replay()
    same = torch.equal(logits.float(), eager)

    def timed(run, n):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for _ in range(3):
            run()
        begin.record()
        for _ in range(n):
            run()
        end.record()
        end.synchronize()
        return begin.elapsed_time(end) / n * 1e3

    result = dict(prompt_us=timed(lambda: decoder(prompt), 5), step_us=timed(graph.replay, a.steps), error=error, graph_equals_eager=same,
                  finite=bool(torch.isfinite(first).all()) and bool((start < a.vocab).all()), status=b2q._lib.device_status())
    print("prompt of %d: %.0f us   step: %.0f us   error against unquantised floats %.2e   graph == eager: %s"
          % (a.prompt, result["prompt_us"], result["step_us"], error, same))
    return result


if __name__ == "__main__":
    main()
