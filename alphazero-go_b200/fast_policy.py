"""A fast policy in 4 bits: a small fully connected network from a position's
planes to move logits, its layers 4-bit microscaled products, its moves drawn
by the sampler, everything on the device.

The residual network answers well but costs a tower per position; a fast
policy plays a position out to its end, or fills in where a move must come at
once. This one is fitted to a teacher's logits: random hidden layers and an
output layer solved for by ridge regression in float32, then all three laid
out in 4 bits.

    teacher = azb200.CudaInference(desc, params, buffers, 256, 0, azb200.BF16)
    policy = FastPolicy.fit(teacher, positions)
    moves, logprob = policy.play(planes, noise, legal, temperature=0.8, top_k=40, top_p=0.95)
    python alphazero-go_b200/fast_policy.py        # fits one to a synthetic teacher and reports
"""
from __future__ import annotations

import numpy as np
import torch

import azb200
import azb_ops


class FastPolicy:
    """planes [B][planes * area] -> logits [B][area + 1]: relu(W1 x + b1),
    relu(W2 h + b2), W3 h + b3, the weights in 4 bits."""

    def __init__(self, weights, biases):
        """weights: three matrices [out, in]; biases: three vectors [out] (float32, on one GPU)."""
        self.layers = [(azb_ops.mx4_quantise(w), b.float().contiguous()) for w, b in zip(weights, biases)]

    @classmethod
    def fit(cls, teacher: azb200.CudaInference, positions: np.ndarray, hidden: int = 1024, ridge: float = 1e-2,
            seed: int = 1) -> "FastPolicy":
        """Fits the output layer to the teacher's logits on `positions`
        ([N][planes][area] float32), passed through the teacher in batches."""
        d = teacher.desc
        g = torch.Generator(device="cuda").manual_seed(seed)
        sizes = [(hidden, d.planes * d.area), (hidden, hidden)]
        weights = [torch.randn(o, i, generator=g, device="cuda") * (2.0 / i) ** 0.5 for o, i in sizes]
        biases = [torch.randn(o, generator=g, device="cuda") * 0.1 for o, _ in sizes]
        policy = cls(weights, biases)
        x = torch.as_tensor(positions.reshape(len(positions), -1), device="cuda")
        h = policy._hidden(x).double()
        target = np.concatenate([teacher.infer(positions[i:i + teacher.max_batch])[0]
                                 for i in range(0, len(positions), teacher.max_batch)])
        h1 = torch.cat([h, torch.ones(len(h), 1, dtype=h.dtype, device="cuda")], 1)
        gram = h1.t() @ h1
        gram += ridge * gram.diagonal().mean() * torch.eye(len(gram), dtype=h.dtype, device="cuda")
        w = torch.linalg.solve(gram, h1.t() @ torch.as_tensor(target, device="cuda").double()).float()
        policy.layers.append((azb_ops.mx4_quantise(w[:-1].t().contiguous()), w[-1].contiguous()))
        return policy

    def _hidden(self, x: torch.Tensor) -> torch.Tensor:
        for w, b in self.layers[:2]:
            x = azb_ops.mx4_product(x, w, bias=b, relu=True, dtype=torch.bfloat16)
        return x

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        w, b = self.layers[2]
        return azb_ops.mx4_product(self._hidden(x), w, bias=b, dtype=torch.float32)

    def play(self, x: torch.Tensor, noise: torch.Tensor, legal: torch.Tensor | None = None, **settings):
        """(moves, logprob) for encoded positions on the GPU; settings as azb_ops.sample_moves takes them."""
        return azb_ops.sample_moves(self.logits(x), noise, legal=legal, **settings)

    def nbytes(self) -> int:
        return sum(w.nbytes() + 4 * b.numel() for w, b in self.layers)


def main() -> None:
    desc = azb200.NetDesc(9, 1, 4, 64, 64, 0)
    params, buffers = azb200.synth_network(desc, 7)
    train, held_out = azb200.synth_positions(desc, 1, 8192), azb200.synth_positions(desc, 2, 1024)
    with azb200.CudaInference(desc, params, buffers, 256, 0, azb200.BF16) as teacher:
        policy = FastPolicy.fit(teacher, train)
        best = np.concatenate([teacher.infer(held_out[i:i + 256])[0] for i in range(0, 1024, 256)])
    x = torch.as_tensor(held_out.reshape(1024, -1), device="cuda")
    legal = torch.ones(1024, desc.actions, dtype=torch.bool, device="cuda")
    legal[:, :-1] = x.view(1024, desc.planes, desc.area)[:, :2].sum(1) == 0      # empty points, and the pass
    noise = torch.rand(1024, desc.actions, device="cuda")
    logits = policy.logits(x)
    t = torch.as_tensor(best, device="cuda")
    corr = torch.corrcoef(torch.stack([(v - v.mean(1, keepdim=True)).flatten() for v in (logits, t)]))[0, 1]
    policy.play(x, noise, legal, temperature=0.8, top_k=20, top_p=0.95)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moves, logprob = policy.play(x, noise, legal, temperature=0.8, top_k=20, top_p=0.95)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    graph.replay()
    start.record()
    for _ in range(100):
        graph.replay()
    end.record()
    azb_ops.check(0)
    print(f"fast policy: {policy.nbytes() / 1024:.0f} KiB, correlation with the teacher's logits {corr:.3f} on "
          f"held-out positions, {start.elapsed_time(end) * 10:.1f} us for 1024 positions (planes to moves), "
          f"mean logprob {logprob.mean():.2f}, all legal {bool(legal.gather(1, moves.clamp(min=0)[:, None]).all())}")


if __name__ == "__main__":
    main()
