"""Patches with their places through experts that learn: the layer entries
(hip_layers.h) of a training step, and of acting on the same weights in 8 bits.

  places    a learned vector of each of a camera's 64 patches, four cameras
            (256 entries), added to the patches' planes; black patches have none
  router    logits, two of eight experts a token, none for a black patch; the
            choices in the experts' order
  rows      the tokens copied into that order
  experts   up with SiLU, down: products per expert, torch's while learning, in
            8-bit integers while acting
  sum       token + its experts' rows with the routing's weights

The planes and weights are random.  `learn` returns the gradients of everything
that the step reads; the choice of the experts is held fixed.

    python examples/trained_experts.py [environments]
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from turbinator_c_amd import layers  # noqa: E402

PLACES, WIDTH, HIDDEN, EXPERTS, TOP = 256, 256, 512, 8, 2
SCALE = 0.5  # of a place's vector
F32, BF16 = layers.DTYPES["f32"], layers.DTYPES["bf16"]
SILU, NONE = layers.ACTS["silu"], layers.ACTS["none"]
SOFTMAX = layers.SCORES["softmax"]


def done(status: int) -> None:
    if status != 1:
        raise RuntimeError("a layer entry refused its arguments")


def space(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def row(x: torch.Tensor) -> int:
    return x.stride(0) * x.element_size()


class EightBit:
    """`rows` rows of k as codes and scales."""

    def __init__(self, rows: int, k: int):
        self.rows, self.k = rows, k
        self.codes = space(rows, layers.int8_padded(k), dtype=torch.int8)
        self.scales = space(rows)

    def take(self, x: torch.Tensor, stream) -> "EightBit":
        done(layers.int8_quantise_device(x, row(x), self.codes, self.scales, self.rows, self.k,
                                         layers.DTYPES[x.dtype], stream))
        return self


class TrainedExperts:
    def __init__(self, environments: int, dtype=torch.bfloat16, seed: int = 1):
        self.dtype, self.code = dtype, layers.DTYPES[dtype]
        self.tokens = environments * PLACES
        rng = torch.Generator().manual_seed(seed)

        def random(*shape, scale):
            return (torch.randn(*shape, generator=rng) * scale).to(dtype).cuda()

        self.table = random(PLACES, WIDTH, scale=1.0)
        self.router = random(WIDTH, EXPERTS, scale=0.2)
        self.up = random(EXPERTS, HIDDEN, WIDTH, scale=WIDTH ** -0.5)
        self.down = random(EXPERTS, WIDTH, HIDDEN, scale=HIDDEN ** -0.5)
        t, rows = self.tokens, self.tokens * TOP
        self.token, self.out = (space(t, WIDTH, dtype=dtype) for _ in range(2))
        self.ids, self.order = (space(t, dtype=torch.int32) for _ in range(2))
        self.ranges = space(PLACES, 2, dtype=torch.int32)
        self.experts, self.positions = (space(t, TOP, dtype=torch.int32) for _ in range(2))
        self.weights, self.dweights = space(t, TOP), space(t, TOP)
        self.offsets = space(EXPERTS + 1, dtype=torch.int32)
        self.row_token = space(rows, dtype=torch.int32)
        self.rows, self.part, self.drows, self.dpart = (space(rows, WIDTH, dtype=dtype)
                                                        for _ in range(4))
        self.dlogits = space(t, EXPERTS, dtype=dtype)
        self.dtoken, self.dtable = space(t, WIDTH, dtype=dtype), space(PLACES, WIDTH)
        need = max(layers.expert_order_workspace_bytes(t, EXPERTS, TOP),
                   layers.embed_order_workspace_bytes(t, PLACES),
                   layers.embed_backward_workspace_bytes(t, PLACES, WIDTH))
        self.workspace = space(need, dtype=torch.uint8)
        self.token8, self.hidden8 = EightBit(t, WIDTH), EightBit(rows, HIDDEN)
        self.hidden = space(rows, HIDDEN, dtype=dtype)
        self.up8, self.down8 = EightBit(EXPERTS * HIDDEN, WIDTH), EightBit(EXPERTS * WIDTH, HIDDEN)
        self.freeze()

    def freeze(self) -> None:
        """The experts' matrices in 8 bits, after each change of them."""
        stream = torch.cuda.current_stream()
        self.up8.take(self.up.flatten(0, 1), stream)
        self.down8.take(self.down.flatten(0, 1), stream)

    def route(self, planes, valid) -> None:
        stream, t = torch.cuda.current_stream(), self.tokens
        place = torch.arange(t, device="cuda", dtype=torch.int32) % PLACES
        self.ids.copy_(torch.where(valid != 0, place, -1))
        done(layers.embed_device(self.ids, self.table, row(self.table), planes, row(planes), SCALE,
                                 self.token, t, PLACES, WIDTH, self.code, stream))
        self.logits = self.token @ self.router
        done(layers.route_device(self.logits, row(self.logits), None, valid, self.experts,
                                 self.weights, t, EXPERTS, TOP, 1, 1, SOFTMAX, True, 1.0,
                                 self.code, stream))
        done(layers.expert_order_device(self.experts, None, self.offsets, self.row_token,
                                        self.positions, None, self.workspace, t, EXPERTS, TOP,
                                        stream))

    def sum(self) -> torch.Tensor:
        done(layers.expert_sum_device(self.part, row(self.part), self.positions, self.weights,
                                      self.token, row(self.token), self.out, self.tokens, TOP,
                                      WIDTH, self.code, torch.cuda.current_stream()))
        return self.out

    def forward(self, planes, valid) -> torch.Tensor:
        """The tokens with their experts' rows, for planes [tokens, WIDTH]."""
        self.route(planes, valid)
        done(layers.expert_rows_device(self.token, row(self.token), self.offsets, self.positions,
                                       None, self.rows, self.tokens, EXPERTS, TOP, WIDTH,
                                       self.code, torch.cuda.current_stream()))
        self.ends = self.offsets.tolist()
        self.z = []
        self.part.zero_()
        for e, (lo, hi) in enumerate(zip(self.ends, self.ends[1:])):
            z = self.rows[lo:hi] @ self.up[e].T
            self.z.append(z)
            self.part[lo:hi] = torch.nn.functional.silu(z) @ self.down[e].T
        return self.sum()

    def learn(self, dout) -> dict:
        """The gradients for the gradient of forward's result, after it."""
        stream, t = torch.cuda.current_stream(), self.tokens
        done(layers.expert_sum_backward_device(dout, row(dout), self.part, row(self.part),
                                               self.offsets, self.positions, self.weights,
                                               self.dpart, self.dweights, t, EXPERTS, TOP, WIDTH,
                                               self.code, stream))
        dup, ddown = torch.zeros_like(self.up), torch.zeros_like(self.down)
        self.drows.zero_()
        for e, (lo, hi) in enumerate(zip(self.ends, self.ends[1:])):
            z, d = self.z[e].float(), self.dpart[lo:hi]
            s = torch.sigmoid(z)
            ddown[e] = d.T.contiguous() @ (z * s).to(self.dtype)
            dz = (d @ self.down[e]).float() * s * (1 + z * (1 - s))
            dup[e] = dz.to(self.dtype).T.contiguous() @ self.rows[lo:hi]
            self.drows[lo:hi] = dz.to(self.dtype) @ self.up[e]
        done(layers.expert_rows_backward_device(self.drows, row(self.drows), None, 0,
                                                self.positions, None, self.dtoken, None, t, TOP,
                                                WIDTH, self.code, stream))
        done(layers.route_backward_device(self.logits, row(self.logits), self.experts,
                                          self.dweights, self.dlogits, t, EXPERTS, TOP, SOFTMAX,
                                          True, 1.0, self.code, stream))
        dplanes = dout + self.dtoken + self.dlogits @ self.router.T.contiguous()
        done(layers.embed_order_device(self.ids, self.order, self.ranges, self.workspace, t,
                                       PLACES, stream))
        done(layers.embed_backward_device(dplanes, row(dplanes), self.ids, self.order, self.ranges,
                                          SCALE, self.dtable, self.workspace, t, PLACES, WIDTH,
                                          self.code, stream))
        return {"table": self.dtable, "router": self.token.T.contiguous() @ self.dlogits,
                "up": dup, "down": ddown, "planes": dplanes, "weights": self.dweights}

    def act(self, planes, valid) -> torch.Tensor:
        """forward with the experts in 8 bits: launches alone, nothing read back."""
        stream, rows = torch.cuda.current_stream(), self.tokens * TOP
        self.route(planes, valid)
        self.token8.take(self.token, stream)
        done(layers.int8_product_device(self.token8.codes, self.token8.scales, self.tokens,
                                        self.row_token, self.up8.codes, self.up8.scales,
                                        self.offsets, None, None, self.hidden, rows, HIDDEN, WIDTH,
                                        EXPERTS, SILU, self.code, stream))
        self.hidden8.take(self.hidden, stream)
        done(layers.int8_product_device(self.hidden8.codes, self.hidden8.scales, rows, None,
                                        self.down8.codes, self.down8.scales, self.offsets, None,
                                        None, self.part, rows, WIDTH, HIDDEN, EXPERTS, NONE,
                                        self.code, stream))
        return self.sum()


def inputs(environments: int, dtype=torch.bfloat16, seed: int = 2):
    """Planes of the patches, and which patches are not black (seven of eight)."""
    rng = torch.Generator().manual_seed(seed)
    tokens = environments * PLACES
    planes = torch.randn(tokens, WIDTH, generator=rng).to(dtype).cuda()
    return planes, (torch.rand(tokens, generator=rng) < 0.875).to(torch.uint8).cuda()


def main() -> None:
    n = int(sys.argv[1]) if len(sys.argv) > 1 else 64
    planes, valid = inputs(n)
    net = TrainedExperts(n)

    def time(call, times=20):
        for _ in range(3):
            call()
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(times):
            call()
        end.record()
        end.synchronize()
        return begin.elapsed_time(end) / times * 1e3

    out = net.forward(planes, valid).clone()
    print(f"{n} environments, {net.tokens} tokens of {WIDTH}, {TOP} of {EXPERTS} experts")
    print(f"rows of each expert: {net.offsets.diff().tolist()}")
    dout = torch.randn_like(out)
    print(f"forward  {time(lambda: net.forward(planes, valid)):8.1f} us")
    print(f"learning {time(lambda: net.learn(dout)):8.1f} us")
    off = (net.act(planes, valid) - out).float().norm() / out.float().norm()
    print(f"acting   {time(lambda: net.act(planes, valid)):8.1f} us, {off:.4f} off the training form")


if __name__ == "__main__":
    main()
