"""A mixture-of-experts MLP with MXFP4 weights and LoRA adapters, as a serving step runs it.

    y = shared(x) + sum_j weight_j expert_j(x),   expert(x) = down (silu(gate x) * (up x))

The routed experts and the shared expert hold MXFP4 weights (4.25 bits a value);
each token's LoRA adapter acts on the shared expert's down projection. Eight
launches a step, three more with MXFP4 activations and one where many tokens route, all on the
caller's stream without a read-back, so the step can be captured in a graph.

    python -m examples.moe_block [tokens ...]
"""

from __future__ import annotations

import sys
import time
from dataclasses import dataclass

import torch

from loraforge_amd.ops import (
    LoraBatch,
    MXFP4Tensor,
    combine_experts,
    expert_linear,
    lora_apply,
    mxfp4_linear,
    quantize_mxfp4,
    route_experts,
)


@dataclass
class MoeBlock:
    router: torch.Tensor  # bf16 [experts, hidden]
    gate_up: MXFP4Tensor  # [experts, 2 inter, hidden]: gate rows, then up rows
    down: MXFP4Tensor  # [experts, hidden, inter]
    shared_gate_up: MXFP4Tensor  # [2 shared, hidden]
    shared_down: MXFP4Tensor  # [hidden, shared]
    top_k: int
    # From this many tokens on activations are quantised too, which makes the products
    # four times as fast at most; a decode batch is bound by the weights' bytes either way.
    quantize_from: int | None = None

    @classmethod
    def from_bf16(cls, router, gate_up, down, shared_gate_up, shared_down, top_k, quantize_from=None) -> "MoeBlock":
        packed = [quantize_mxfp4(w) for w in (gate_up, down, shared_gate_up, shared_down)]
        return cls(router, *packed, top_k, quantize_from)

    def __call__(self, x: torch.Tensor, lora: LoraBatch | None = None) -> torch.Tensor:
        quantized = self.quantize_from is not None and x.shape[0] >= self.quantize_from
        act = quantize_mxfp4 if quantized else (lambda t: t)
        r = route_experts(x @ self.router.T, self.top_k)
        xa = act(x)
        h = expert_linear(xa, self.gate_up, r.offsets, tokens=r.tokens, swiglu=True)
        rows = expert_linear(act(h), self.down, r.offsets)
        s = mxfp4_linear(xa, self.shared_gate_up, swiglu=True)
        y = mxfp4_linear(act(s), self.shared_down)
        if lora is not None:
            lora_apply(s, y, lora)
        return combine_experts(rows, r.positions, r.weights, base=y, out=y)


def adapters(count: int, rank: int, shared: int, hidden: int, tokens: int, device, generator) -> LoraBatch:
    """`count` random adapters of one rank on the shared down projection, dealt to the tokens in turn."""
    stride = 1 << (rank - 1).bit_length()
    integers = dict(dtype=torch.int32, device=device)
    return LoraBatch.from_padded(
        (torch.randn(count, rank, shared, generator=generator) * shared**-0.5).bfloat16().to(device),
        (torch.randn(count * hidden * stride, generator=generator) * 0.05).bfloat16().to(device),
        b_offsets=torch.arange(count, dtype=torch.int64, device=device) * (hidden * stride),
        b_strides=torch.full((count,), stride, **integers),
        ranks=torch.full((count,), rank, **integers),
        scales=torch.full((count,), 2.0, dtype=torch.float32, device=device),
        token_slots=torch.arange(tokens, **integers) % count,
        slice_offsets=torch.tensor([0, hidden], **integers),
        max_rank=rank,
    )


def random_block(hidden, inter, shared, experts, top_k, device, generator, quantize_from=None) -> MoeBlock:
    def w(*shape):
        return (torch.randn(*shape, generator=generator) * shape[-1] ** -0.5).bfloat16().to(device)

    return MoeBlock.from_bf16(w(experts, hidden), w(experts, 2 * inter, hidden), w(experts, hidden, inter),
                              w(2 * shared, hidden), w(hidden, shared), top_k, quantize_from)


def capture(block: MoeBlock, x, lora=None):
    """A graph of one step and its output; new tokens go into ``x`` before each replay."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(x, lora)  # (lora_apply makes its workspace for the stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = block(x, lora)
    return graph, y


def main(sizes) -> None:
    device, g = torch.device("cuda:0"), torch.Generator().manual_seed(0)
    hidden, inter, shared, experts, top_k = 4096, 1024, 2048, 64, 4
    block = random_block(hidden, inter, shared, experts, top_k, device, g, quantize_from=512)
    for tokens in sizes:
        x = torch.randn(tokens, hidden, generator=g).bfloat16().to(device)
        lora = adapters(8, 16, shared, hidden, tokens, device, g)
        graph, y = capture(block, x, lora)
        graph.replay()
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(20):
            graph.replay()
        torch.cuda.synchronize()
        print(f"{tokens:6d} tokens  {(time.perf_counter() - start) / 20 * 1e6:9.1f} us a step  |y| {y.float().norm():.4g}", flush=True)


if __name__ == "__main__":
    main([int(a) for a in sys.argv[1:]] or [1, 16, 64, 512, 4096])
